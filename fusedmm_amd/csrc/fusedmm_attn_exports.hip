// Entry points of the attention family (include/fusedmm_amd.h): what they check, and how a call becomes launches.
// Built once per (INDEXTYPE, VALUETYPE) as the other entry points are; VALUETYPE plays no part, INDEXTYPE is the width of
// the index arrays.
#include <algorithm>
#include <cmath>
#include <new>

#include "fusedmm_attn.hpp"

#ifndef INDEXTYPE
#error "compile with -DINDEXTYPE=int32_t or -DINDEXTYPE=int64_t"
#endif
#ifdef DREAL
#define VALUETYPE double
#else
#define VALUETYPE float
#endif
#pragma GCC visibility push(default)
#include "../../include/fusedMM.h"
#include "../../include/fusedmm_amd.h"
#pragma GCC visibility pop

namespace {

using namespace fmm_attn;
typedef fusedMM_attn_desc Desc;

static_assert(kOk == FUSEDMM_SUCCESS_RETURN && kFail == FUSEDMM_FAIL_RETURN && kNoMem == FUSEDMM_NOT_ENOUGH_MEM && kNoImpl == FUSEDMM_NO_OPT_IMPL, "");
static_assert(kF32 == FUSEDMM_TYPE_F32 && kF16 == FUSEDMM_TYPE_F16 && kBF16 == FUSEDMM_TYPE_BF16, "");

constexpr int64_t kMaxTokens = (int64_t)1 << 20;
constexpr int64_t kMaxSlots = (int64_t)1 << 44;   // of a serving call

int refuse(const char *who, const char *why)
{
   ATTN_LOG("%s: %s", who, why);
   return kFail;
}

int element_bytes(const Desc &d) { return d.type == FUSEDMM_TYPE_F32 ? 4 : 2; }
int64_t align256(int64_t v) { return (v + 255) & ~(int64_t)255; }

// the sizes that every call needs; *dc is the width class
int check_sizes(const char *who, const Desc *d, int *dc)
{
   if (!d) return refuse(who, "no descriptor");
   if (d->type < FUSEDMM_TYPE_F32 || d->type > FUSEDMM_TYPE_BF16) return refuse(who, "unknown element type");
   if (d->maps != 1 && d->maps != 2) return refuse(who, "maps is 1 or 2");
   if (d->m < 0 || d->n < 0) return refuse(who, "negative size");
   if (d->kv_heads < 1 || d->d < 1 || d->dv < 1) return refuse(who, "kv_heads, d and dv are at least 1");
   *dc = width_class(d->d, d->dv, d->maps);
   if (!*dc)
   {
      ATTN_LOG("%s: no kernel for d = %d, dv = %d with %d map(s)", who, d->d, d->dv, d->maps);
      return kNoImpl;
   }
   return kOk;
}

int check_heads(const char *who, const Desc &d)
{
   if (d.heads < 1 || d.heads % d.kv_heads) return refuse(who, "heads is a positive multiple of kv_heads");
   return kOk;
}

// (the softmax takes a score factor of NaN or zero for its least positive one)
int check_scale(const char *who, const Desc &d) { return std::isfinite(d.scale) ? kOk : refuse(who, "scale is not a finite number"); }

bool strides_ok(int64_t ld, int64_t hd)
{
   return ld >= 0 && hd >= 0 && ld < ((int64_t)1 << 29) && hd < ((int64_t)1 << 48);   // a row's bytes fit 32 bits
}

// (row, head) pieces of `width` elements that do not overlap: packed rows, or whole heads.  (In 128 bits: 2^31 heads of a
// stride of 2^47 are past 64.)
bool apart(int64_t ld, int64_t hd, int64_t rows, int64_t heads, int64_t width)
{
   typedef __int128 wide;
   const bool rows_outer = (heads == 1 || hd >= width) && (rows <= 1 || ld >= (wide)(heads - 1) * hd + width);
   const bool heads_outer = (rows <= 1 || ld >= width) && (heads == 1 || hd >= (wide)(rows > 0 ? rows - 1 : 0) * ld + width);
   return rows_outer || heads_outer;
}

bool lines_up(const void *p, int64_t ld, int64_t hd, int bytes) { return ((uintptr_t)p & 15) == 0 && (ld * bytes) % 16 == 0 && (hd * bytes) % 16 == 0; }

// Device memory of the current device.  (A null pointer where one is needed is refused by the caller.)
int check_pointers(const char *who, const void *const *ptrs, int count)
{
   int dev = 0;
   ATTN_HIP(hipGetDevice(&dev));
   for (int i = 0; i < count; i++)
   {
      if (!ptrs[i]) continue;
      hipPointerAttribute_t a;
      if (hipPointerGetAttributes(&a, ptrs[i]) != hipSuccess)
      {
         (void)hipGetLastError();
         return refuse(who, "an operand is not device memory");
      }
      if (a.type != hipMemoryTypeDevice && a.type != hipMemoryTypeManaged) return refuse(who, "an operand is not device memory");
      if (a.type == hipMemoryTypeDevice && a.device != dev) return refuse(who, "an operand lives on another device than the current one");
   }
   return kOk;
}

const Plan *as_plan(const void *p)
{
   const Plan *plan = (const Plan *)p;
   return plan && plan->magic == kPlanMagic ? plan : nullptr;
}

PlanSizes sizes_of(const Plan &p) { return {p.view.n_units, p.view.n_joins, p.tiles, p.view.block_rows}; }

// plan (and plan_t, with which a backward pass is asked for) against the descriptor
int check_plans(const char *who, const Desc &d, int dc, const void *plan, const void *plan_t, bool need_t)
{
   const Plan *p = as_plan(plan), *t = as_plan(plan_t);
   if (!p || (need_t && !t) || (plan_t && !t)) return refuse(who, "no plan, or one that was destroyed");
   if (p->rows != d.m || p->cols != d.n) return refuse(who, "the plan is of a pattern of another size");
   if (t && (t->rows != d.n || t->cols != d.m)) return refuse(who, "the second plan is not of the transposed pattern's size");
   if (t && t->device != p->device) return refuse(who, "the plans belong to different devices");
   const int w = dc * d.maps;
   if (!forward_fits(sizes_of(*p), d.heads, w) || !pack_fits(d.heads) || (t && !backward_fits(sizes_of(*p), sizes_of(*t), d.heads, d.kv_heads, w)))
      return refuse(who, "too many rows and heads for one call");
   return kOk;
}

int check_device(const char *who, const void *plan)
{
   int dev = 0;
   ATTN_HIP(hipGetDevice(&dev));
   return as_plan(plan)->device == dev ? kOk : refuse(who, "the plan belongs to another device than the current one");
}

bool whole_chunks(const Desc &d)
{
   const int epl = 16 / element_bytes(d);
   return d.d % epl == 0 && d.dv % epl == 0;
}

// The tensors whose rows a kernel gathers.  Where their sizes or strides keep rows off 16 bytes they are laid out anew in the
// workspace, once per call: training with 5 columns that all of 1808 rows name, 16 heads, two maps of 38 and 75 bf16
// features, 185 us instead of 435.  (A pointer alone that is off, which the descriptor does not tell, is not.)
struct Tensors {
   const void *a = nullptr, *b = nullptr;
   int64_t rows = 0, lda = 0, ha = 0, ldb = 0, hb = 0;
   int heads = 0;
};
Tensors keys_values(const Desc &d, const void *k, const void *v) { return {k, v, d.n, d.ldk, d.hdk, d.ldv, d.hdv, d.kv_heads}; }
Tensors queries_gradients(const Desc &d, const void *q, const void *dout) { return {q, dout, d.m, d.ldq, d.hdq, d.ldo, d.hdo, d.heads}; }

bool packs(const Desc &d, const Tensors &t)
{
   const int bytes = element_bytes(d);
   return t.rows > 0 && (!whole_chunks(d) || (t.lda * bytes) % 16 || (t.ha * bytes) % 16 || (t.ldb * bytes) % 16 || (t.hb * bytes) % 16);
}
int64_t pack_bytes(const Desc &d, const Tensors &t, int dc) { return packs(d, t) ? 2 * t.rows * t.heads * dc * d.maps * element_bytes(d) : 0; }

// how the kernels find them; copies them to `to` where they are to be packed
int gather_from(const Desc &d, const Tensors &t, int dc, void *to, hipStream_t s, Gathered *g)
{
   const int bytes = element_bytes(d), w = dc * d.maps;
   if (!packs(d, t))
   {
      const bool vec = whole_chunks(d) && lines_up(t.a, t.lda, t.ha, bytes) && lines_up(t.b, t.ldb, t.hb, bytes);
      *g = Gathered{t.a, t.b, t.ha, t.hb, (int32_t)(t.lda * bytes), (int32_t)(t.ldb * bytes), d.d, d.dv, vec, vec && d.d == dc && d.dv == w};
      return kOk;
   }
   void *to_b = (unsigned char *)to + t.rows * t.heads * w * bytes;
   *g = Gathered{to, to_b, t.rows * w, t.rows * w, w * bytes, w * bytes, dc, w, 1, 1};
   PackParams p{t.a, t.b, to, to_b, t.rows, t.lda, t.ha, t.ldb, t.hb, t.heads, d.d, d.dv, dc, w * bytes / 16, 0};
   p.per_head = (int32_t)pack_per_head(t.rows, t.heads, p.chunks);
   return d.type == FUSEDMM_TYPE_F32 ? launch_pack_f32(p, s) : d.type == FUSEDMM_TYPE_F16 ? launch_pack_f16(p, s) : launch_pack_bf16(p, s);
}

struct Layout {   // of a workspace, in bytes
   int64_t stats = 0, dlam = 0, part = 0, pack = 0, total = 0;
};

Layout forward_layout(const Desc &d, const Plan &p, int dc)
{
   Layout l;
   l.pack = align256(p.parts * d.heads * forward_part(dc, d.maps, p.view.block_rows) * 4);
   l.total = l.pack + pack_bytes(d, keys_values(d, nullptr, nullptr), dc);
   return l;
}

Layout backward_layout(const Desc &d, const Plan &p, const Plan &t, int dc)
{
   Layout l;
   l.dlam = align256(d.m * d.heads * d.maps * 8);
   l.part = l.dlam + (d.maps == 2 ? align256((int64_t)p.view.n_units * (p.view.block_rows / 16) * d.heads * 4) : 0);
   l.pack = l.part + align256(std::max(p.parts * d.heads * dq_part(dc, d.maps, p.view.block_rows), t.parts * d.kv_heads * dkv_part(dc, d.maps, t.view.block_rows)) * 4);
   // (one after the other)
   l.total = l.pack + std::max(pack_bytes(d, keys_values(d, nullptr, nullptr), dc), pack_bytes(d, queries_gradients(d, nullptr, nullptr), dc));
   return l;
}

int check_work(const char *who, const void *work, int64_t have, int64_t need)
{
   if (need <= 0) return kOk;
   if (!work || have < need)
   {
      ATTN_LOG("%s: the workspace has %lld bytes, %lld are needed", who, (long long)(work ? have : 0), (long long)need);
      return kNoMem;
   }
   if ((uintptr_t)work & 15) return refuse(who, "the workspace is not 16-byte aligned");
   return kOk;
}

Params base_params(const Desc &d, const Plan &plan)
{
   Params p{};
   p.plan = plan.view;
   p.m = d.m;
   p.n = d.n;
   p.heads = d.heads;
   p.kv_heads = d.kv_heads;
   p.group = d.heads / d.kv_heads;
   p.d = d.d;
   p.dv = d.dv;
   p.scale = d.scale;
   p.ldq = d.ldq;
   p.hdq = d.hdq;
   p.ldk = d.ldk;
   p.hdk = d.hdk;
   p.ldv = d.ldv;
   p.hdv = d.hdv;
   p.ldo = d.ldo;
   p.hdo = d.hdo;
   return p;
}

bool inputs_ok(const Desc &d)
{
   return strides_ok(d.ldq, d.hdq) && strides_ok(d.ldk, d.hdk) && strides_ok(d.ldv, d.hdv) && strides_ok(d.ldo, d.hdo);
}

// ---- serving form ----

// Slots of a piece, over all key heads.  In the tensors' own type about 1024 workgroups, two rounds of the 2 that a CU holds:
// a ragged batch takes 125 us, with 768 or 2048 workgroups 129 us.  In 4 bits about 768, one round of the 3 that a CU holds: two
// rows of 200k slots take 37 us, with 1024 workgroups 42 us, a ragged batch 149 and 146 us.  Not under 256 slots (two
// tiles per wave), not over 8192.
int64_t piece_slots(int64_t nnz, int64_t columns, bool kv4)
{
   const int64_t want = std::min<int64_t>(nnz, 8192 * 1024) * columns / (kv4 ? 768 : 1024);   // (longer lists reach 8192 anyhow)
   return (std::min<int64_t>(std::max<int64_t>(want, 256), 8192) + 127) / 128 * 128;
}

struct RowsPlan {
   bool fits = false;   // in a launch, and its sizes in 64 bits
   int passes = 0;
   int64_t piece = 0, cap = 0, table = 0, total = 0;   // table: byte offset behind the partial sums
};

RowsPlan rows_plan(const Desc &d, int64_t nnz, int dc, bool kv4)
{
   RowsPlan r;
   const int hp = 16 / d.maps, group = d.heads / d.kv_heads;
   r.passes = (group + hp - 1) / hp;
   const int64_t columns = (int64_t)d.kv_heads * r.passes;
   if (d.m > INT32_MAX || nnz > kMaxSlots || !rows_fit(d.m, d.m, columns, d.heads)) return r;
   r.piece = piece_slots(nnz, columns, kv4);
   const bool cut = nnz > r.piece && d.m > 0;
   const int64_t most = (cut ? nnz / r.piece : 0) + d.m;
   r.fits = rows_fit(most, d.m, columns, d.heads);
   if (!r.fits || !cut) return r;
   r.cap = most;
   r.table = align256(r.cap * columns * 16 * (dc * d.maps + kPartExtra) * 4);
   r.total = r.table + (d.m > kTableRows ? (d.m + 2) * 8 : 0);
   return r;
}

int rows_common(const char *who, bool kv4, const Desc *d, int64_t nnz, const void *indx, const void *pntrb, const void *pntre, const void *q, const float *lambda,
                void *o, void *work, int64_t work_bytes, int *dc, RowsParams *p)
{
   int st = check_sizes(who, d, dc);
   if (st) return st;
   st = check_heads(who, *d);
   if (!st) st = check_scale(who, *d);
   if (st) return st;
   if (nnz < 0) return refuse(who, "negative nnz");
   if (d->n > INT32_MAX) return refuse(who, "n is at most 2^31 - 1");
   if (!inputs_ok(*d)) return refuse(who, "a stride is negative or too large");
   if (!apart(d->ldo, d->hdo, d->m, d->heads, d->dv)) return refuse(who, "the rows of o overlap");
   const RowsPlan r = rows_plan(*d, nnz, *dc, kv4);
   if (!r.fits) return refuse(who, "too many rows, slots and heads for one call");
   if (d->m == 0) return kOk;
   if (!q || !o || !pntrb || !pntre || (nnz > 0 && !indx) || (d->maps == 2 && !lambda)) return refuse(who, "a pointer is null");
   st = check_work(who, work, work_bytes, r.total);
   if (st) return st;
   const int bytes = element_bytes(*d);
   *p = RowsParams{};
   p->m = d->m;
   p->n = d->n;
   p->heads = d->heads;
   p->kv_heads = d->kv_heads;
   p->group = d->heads / d->kv_heads;
   p->d = d->d;
   p->dv = d->dv;
   p->passes = r.passes;
   p->scale = d->scale;
   p->index_bytes = (int)sizeof(INDEXTYPE);
   p->indx = indx;
   p->pntrb = pntrb;
   p->pntre = pntre;
   p->q = q;
   p->ldq = d->ldq;
   p->hdq = d->hdq;
   p->ldk = d->ldk;
   p->hdk = d->hdk;
   p->ldv = d->ldv;
   p->hdv = d->hdv;
   p->ldo = d->ldo;
   p->hdo = d->hdo;
   p->vec_q = whole_chunks(*d) && lines_up(q, d->ldq, d->hdq, bytes);
   p->lambda = lambda;
   p->out = o;
   p->out_type = d->type;
   p->piece = r.piece;
   p->cap = r.cap;
   p->part = (float *)work;
   p->table = (int64_t *)((unsigned char *)work + r.table);
   return kOk;
}

// ---- 4-bit cache ----

int64_t record_bytes(int maps, int d, int dv)
{
   const int64_t w = (int64_t)maps * d + dv;
   return (w / 2 + w / 16 + 15) / 16 * 16;
}

int check_cache(const char *who, const Desc &d, const void *cache, int64_t ldc, int64_t hdc, bool written)
{
   if (d.d % 32 || d.dv % 32)
   {
      ATTN_LOG("%s: d and dv of a 4-bit cache are multiples of 32", who);
      return kNoImpl;
   }
   if (!strides_ok(ldc, hdc) || ldc % 16 || hdc % 16 || ((uintptr_t)cache & 15)) return refuse(who, "the records of the cache are not 16-byte aligned");
   if (written && !apart(ldc, hdc, d.n, d.kv_heads, record_bytes(d.maps, d.d, d.dv))) return refuse(who, "the records of the cache overlap");
   return kOk;
}

int kv4_common(const char *who, const Desc *desc, int64_t tokens, const void *slots, const void *k, const void *v, const void *cache, int64_t ldc, int64_t hdc,
               bool write, Kv4Params *p)
{
   int dc;
   if (!desc) return refuse(who, "no descriptor");
   Desc own = *desc;
   own.m = 0;   // not read
   const Desc *d = &own;
   int st = check_sizes(who, d, &dc);
   if (st) return st;
   st = check_cache(who, *d, cache, ldc, hdc, write);
   if (st) return st;
   if (tokens < 0) return refuse(who, "negative number of tokens");
   if (write && tokens > kMaxTokens) return refuse(who, "more than 2^20 tokens in one call");
   if (!strides_ok(d->ldk, d->hdk) || !strides_ok(d->ldv, d->hdv)) return refuse(who, "a stride is negative or too large");
   if (!write && (!apart(d->ldk, d->hdk, tokens, d->kv_heads, (int64_t)d->maps * d->d) || !apart(d->ldv, d->hdv, tokens, d->kv_heads, d->dv)))
      return refuse(who, "the rows of k or v overlap");
   const int64_t words = ((int64_t)d->maps * d->d + d->dv) / 8;
   if (d->n > INT32_MAX) return refuse(who, "n is at most 2^31 - 1");
   if (words * d->kv_heads > INT32_MAX / 32) return refuse(who, "too many key heads");
   if (tokens == 0) return kOk;
   if (!slots || !k || !v || !cache) return refuse(who, "a pointer is null");
   const void *ptrs[4] = {slots, k, v, cache};
   st = check_pointers(who, ptrs, 4);
   if (st) return st;
   *p = Kv4Params{};
   p->tokens = tokens;
   p->n = d->n;
   p->kv_heads = d->kv_heads;
   p->k_width = d->maps * d->d;
   p->v_width = d->dv;
   p->index_bytes = (int)sizeof(INDEXTYPE);
   p->slots = slots;
   p->ldk = d->ldk;
   p->hdk = d->hdk;
   p->ldv = d->ldv;
   p->hdv = d->hdv;
   const int bytes = element_bytes(*d);
   p->vec = lines_up(k, d->ldk, d->hdk, bytes) && lines_up(v, d->ldv, d->hdv, bytes);
   p->ldc = ldc;
   p->hdc = hdc;
   return kOk;
}

}  // namespace

extern "C" {

int fusedMM_attn_plan_create(const INDEXTYPE m, const INDEXTYPE n, const INDEXTYPE nnz, const INDEXTYPE *indx, const INDEXTYPE *pntrb, const INDEXTYPE *pntre,
                             void *stream, void **plan)
{
   const char *who = "fusedMM_attn_plan_create";
   if (!plan) return refuse(who, "no place for the plan");
   *plan = nullptr;
   if (m < 0 || n < 0 || nnz < 0 || (int64_t)m > kMaxPlanCols || (int64_t)n > kMaxPlanCols) return refuse(who, "m and n are from 0 to 2^26 - 1, nnz is not negative");
   if (m > 0 && (!pntrb || !pntre || (nnz > 0 && !indx))) return refuse(who, "a pointer is null");
   hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
   ATTN_HIP(hipStreamIsCapturing((hipStream_t)stream, &status));
   if (status != hipStreamCaptureStatusNone) return refuse(who, "a plan waits for the GPU and cannot be made while its stream is captured");
   if (m > 0)
   {
      const void *ptrs[3] = {indx, pntrb, pntre};
      const int st = check_pointers(who, ptrs, 3);
      if (st) return st;
   }
   Plan *p = nullptr;
   int st = kNoMem;
   try
   {
      p = new Plan;
      st = plan_create(p, m, n, nnz, indx, pntrb, pntre, (int)sizeof(INDEXTYPE), (hipStream_t)stream);
   }
   catch (const std::bad_alloc &)
   {
      ATTN_LOG("%s: out of host memory", who);
      st = kNoMem;
   }
   if (st)
   {
      if (p) plan_release(p);
      delete p;
      return st;
   }
   *plan = p;
   return kOk;
}

int fusedMM_attn_plan_destroy(void *plan)
{
   if (!plan) return kOk;
   if (!as_plan(plan)) return refuse("fusedMM_attn_plan_destroy", "not a plan");
   Plan *p = (Plan *)plan;
   plan_release(p);
   delete p;
   return kOk;
}

int64_t fusedMM_attn_workspace(const fusedMM_attn_desc *desc, const void *plan, const void *plan_t)
{
   const char *who = "fusedMM_attn_workspace";
   int dc;
   if (check_sizes(who, desc, &dc) || check_heads(who, *desc) || check_plans(who, *desc, dc, plan, plan_t, false)) return -1;
   int64_t need = forward_layout(*desc, *as_plan(plan), dc).total;
   if (plan_t) need = std::max(need, backward_layout(*desc, *as_plan(plan), *as_plan(plan_t), dc).total);
   return need;
}

int fusedMM_attn_forward(const fusedMM_attn_desc *desc, const void *plan, const void *q, const void *k, const void *v, const float *lambda, void *o, void *o2,
                         float *lse, void *work, int64_t work_bytes, void *stream)
{
   const char *who = "fusedMM_attn_forward";
   int dc;
   int st = check_sizes(who, desc, &dc);
   if (!st) st = check_heads(who, *desc);
   if (!st) st = check_scale(who, *desc);
   if (!st) st = check_plans(who, *desc, dc, plan, nullptr, false);
   if (st) return st;
   const Desc &d = *desc;
   if (!inputs_ok(d)) return refuse(who, "a stride is negative or too large");
   if (!apart(d.ldo, d.hdo, d.m, d.heads, d.dv)) return refuse(who, "the rows of o overlap");
   if (d.m == 0) return kOk;
   if (!q || !o || (d.n > 0 && (!k || !v)) || (d.maps == 2 && !lambda)) return refuse(who, "a pointer is null");
   const Layout l = forward_layout(d, *as_plan(plan), dc);
   st = check_work(who, work, work_bytes, l.total);
   if (!st) st = check_device(who, plan);
   const void *ptrs[] = {q, k, v, lambda, o, o2, lse, work};
   if (!st) st = check_pointers(who, ptrs, 8);
   if (st) return st;
   Params p = base_params(d, *as_plan(plan));
   const int bytes = element_bytes(d);
   p.vec = whole_chunks(d) && lines_up(q, d.ldq, d.hdq, bytes) && lines_up(k, d.ldk, d.hdk, bytes) && lines_up(v, d.ldv, d.hdv, bytes) &&
           lines_up(o, d.ldo, d.hdo, bytes) && lines_up(o2, 0, 0, bytes);
   p.q = q;
   p.k = k;
   p.v = v;
   p.lambda = lambda;
   p.out = o;
   p.out2 = d.maps == 2 ? o2 : nullptr;
   p.lse = lse;
   p.part = (float *)work;
   const hipStream_t s = (hipStream_t)stream;
   st = gather_from(d, keys_values(d, k, v), dc, (unsigned char *)work + l.pack, s, &p.gat);
   if (st) return st;
   return d.type == FUSEDMM_TYPE_F32 ? launch_forward_f32(p, dc, d.maps, s)
          : d.type == FUSEDMM_TYPE_F16 ? launch_forward_f16(p, dc, d.maps, s) : launch_forward_bf16(p, dc, d.maps, s);
}

int fusedMM_attn_backward(const fusedMM_attn_desc *desc, const void *plan, const void *plan_t, const void *q, const void *k, const void *v, const float *lambda,
                          const void *o, const void *o2, const float *lse, const void *dout, void *dq, void *dk, void *dv, float *dlambda, void *work,
                          int64_t work_bytes, void *stream)
{
   const char *who = "fusedMM_attn_backward";
   int dc;
   int st = check_sizes(who, desc, &dc);
   if (!st) st = check_heads(who, *desc);
   if (!st) st = check_scale(who, *desc);
   if (!st) st = check_plans(who, *desc, dc, plan, plan_t, true);
   if (st) return st;
   const Desc &d = *desc;
   if (!inputs_ok(d)) return refuse(who, "a stride is negative or too large");
   if (!apart(d.ldq, d.hdq, d.m, d.heads, (int64_t)d.maps * d.d) || !apart(d.ldk, d.hdk, d.n, d.kv_heads, (int64_t)d.maps * d.d) ||
       !apart(d.ldv, d.hdv, d.n, d.kv_heads, d.dv) || !apart(d.ldo, d.hdo, d.m, d.heads, d.dv))
      return refuse(who, "the rows of a tensor overlap, and so would those of its gradient");
   if ((d.m > 0 && (!q || !o || !lse || !dout || !dq)) || (d.n > 0 && (!k || !v || !dk || !dv)) || (d.maps == 2 && (!lambda || (d.m > 0 && !o2))))
      return refuse(who, "a pointer is null");
   const Plan &pp = *as_plan(plan), &pt = *as_plan(plan_t);
   const Layout l = backward_layout(d, pp, pt, dc);
   st = check_work(who, work, work_bytes, l.total);
   if (!st) st = check_device(who, plan);
   const void *ptrs[] = {q, k, v, lambda, o, o2, lse, dout, dq, dk, dv, dlambda, work};
   if (!st) st = check_pointers(who, ptrs, 13);
   if (st) return st;
   Params p = base_params(d, pp);
   const int bytes = element_bytes(d);
   p.vec = whole_chunks(d) && lines_up(q, d.ldq, d.hdq, bytes) && lines_up(k, d.ldk, d.hdk, bytes) && lines_up(v, d.ldv, d.hdv, bytes) &&
           lines_up(o, d.ldo, d.hdo, bytes) && lines_up(dout, 0, 0, bytes) && lines_up(dq, 0, 0, bytes) && lines_up(dk, 0, 0, bytes) &&
           lines_up(dv, 0, 0, bytes);
   p.q = q;
   p.k = k;
   p.v = v;
   p.lambda = lambda;
   p.o = o;
   p.o2 = o2;
   p.lse_in = lse;
   p.dout = dout;
   p.dq = dq;
   p.dk = dk;
   p.dvv = dv;
   p.dlambda = d.maps == 2 ? dlambda : nullptr;
   p.dlam_count = d.m ? (int64_t)pp.view.n_units * (pp.view.block_rows / 16) : 0;
   p.stats = (float *)((unsigned char *)work + l.stats);
   p.dlam_units = (float *)((unsigned char *)work + l.dlam);
   p.part = (float *)((unsigned char *)work + l.part);
   const hipStream_t s = (hipStream_t)stream;
   void *pack = (unsigned char *)work + l.pack;
   if (d.m > 0)
   {
      st = gather_from(d, keys_values(d, k, v), dc, pack, s, &p.gat);
      if (st) return st;
      st = d.type == FUSEDMM_TYPE_F32 ? launch_dq_f32(p, dc, d.maps, s) : d.type == FUSEDMM_TYPE_F16 ? launch_dq_f16(p, dc, d.maps, s) : launch_dq_bf16(p, dc, d.maps, s);
      if (st) return st;
   }
   if (d.n == 0 && !p.dlambda) return kOk;
   p.plan = pt.view;
   st = gather_from(d, queries_gradients(d, q, dout), dc, pack, s, &p.gat);
   if (st) return st;
   return d.type == FUSEDMM_TYPE_F32 ? launch_dkv_f32(p, dc, d.maps, s) : d.type == FUSEDMM_TYPE_F16 ? launch_dkv_f16(p, dc, d.maps, s) : launch_dkv_bf16(p, dc, d.maps, s);
}

int64_t fusedMM_attn_rows_workspace(const fusedMM_attn_desc *desc, const INDEXTYPE nnz)
{
   const char *who = "fusedMM_attn_rows_workspace";
   int dc;
   if (check_sizes(who, desc, &dc) || check_heads(who, *desc)) return -1;
   if (nnz < 0)
   {
      (void)refuse(who, "negative nnz");
      return -1;
   }
   const RowsPlan own = rows_plan(*desc, nnz, dc, false), four = rows_plan(*desc, nnz, dc, true);
   if (!own.fits || !four.fits)
   {
      (void)refuse(who, "too many rows, slots and heads for one call");
      return -1;
   }
   return std::max(own.total, four.total);
}

int fusedMM_attn_rows(const fusedMM_attn_desc *desc, const INDEXTYPE nnz, const INDEXTYPE *indx, const INDEXTYPE *pntrb, const INDEXTYPE *pntre, const void *q,
                      const void *k, const void *v, const float *lambda, void *o, void *work, int64_t work_bytes, void *stream)
{
   const char *who = "fusedMM_attn_rows";
   int dc;
   RowsParams p;
   int st = rows_common(who, false, desc, nnz, indx, pntrb, pntre, q, lambda, o, work, work_bytes, &dc, &p);
   if (st || desc->m == 0) return st;
   if (desc->n > 0 && (!k || !v)) return refuse(who, "a pointer is null");
   const void *ptrs[] = {indx, pntrb, pntre, q, k, v, lambda, o, work};
   st = check_pointers(who, ptrs, 9);
   if (st) return st;
   const int bytes = element_bytes(*desc);
   p.k = k;
   p.v = v;
   p.vec_kv = whole_chunks(*desc) && lines_up(k, desc->ldk, desc->hdk, bytes) && lines_up(v, desc->ldv, desc->hdv, bytes);
   const hipStream_t s = (hipStream_t)stream;
   return desc->type == FUSEDMM_TYPE_F32 ? launch_rows_f32(p, dc, desc->maps, s)
          : desc->type == FUSEDMM_TYPE_F16 ? launch_rows_f16(p, dc, desc->maps, s) : launch_rows_bf16(p, dc, desc->maps, s);
}

int64_t fusedMM_kv4_record_bytes(const int maps, const int d, const int dv)
{
   if ((maps != 1 && maps != 2) || d < 32 || dv < 32 || d % 32 || dv % 32 || !width_class(d, dv, maps)) return -1;
   return record_bytes(maps, d, dv);
}

int fusedMM_kv4_write(const fusedMM_attn_desc *desc, const INDEXTYPE tokens, const INDEXTYPE *slots, const void *k, const void *v, void *cache, int64_t ldc,
                      int64_t hdc, void *stream)
{
   Kv4Params p;
   const int st = kv4_common("fusedMM_kv4_write", desc, tokens, slots, k, v, cache, ldc, hdc, true, &p);
   if (st || tokens == 0) return st;
   p.k = k;
   p.v = v;
   p.cache = (uint8_t *)cache;
   return launch_kv4_write(p, desc->type, (hipStream_t)stream);
}

int fusedMM_kv4_read(const fusedMM_attn_desc *desc, const INDEXTYPE tokens, const INDEXTYPE *slots, const void *cache, int64_t ldc, int64_t hdc, void *k, void *v,
                     void *stream)
{
   Kv4Params p;
   const int st = kv4_common("fusedMM_kv4_read", desc, tokens, slots, k, v, cache, ldc, hdc, false, &p);
   if (st || tokens == 0) return st;
   p.to_k = k;
   p.to_v = v;
   p.cache = (uint8_t *)const_cast<void *>(cache);
   return launch_kv4_read(p, desc->type, (hipStream_t)stream);
}

int fusedMM_attn_rows_kv4(const fusedMM_attn_desc *desc, const INDEXTYPE nnz, const INDEXTYPE *indx, const INDEXTYPE *pntrb, const INDEXTYPE *pntre,
                          const void *q, const void *cache, int64_t ldc, int64_t hdc, const float *lambda, void *o, void *work, int64_t work_bytes, void *stream)
{
   const char *who = "fusedMM_attn_rows_kv4";
   int dc;
   RowsParams p;
   int st = rows_common(who, true, desc, nnz, indx, pntrb, pntre, q, lambda, o, work, work_bytes, &dc, &p);
   if (st) return st;
   if (desc->type == FUSEDMM_TYPE_F32)
   {
      ATTN_LOG("%s: q and o are fp16 or bf16", who);
      return kNoImpl;
   }
   st = check_cache(who, *desc, cache, ldc, hdc, false);
   if (!st && dc * desc->maps == 256 && (desc->d != dc || desc->dv != 256))
   {
      ATTN_LOG("%s: over 128 features a key or value, d is %d and dv 256", who, dc);
      st = kNoImpl;
   }
   if (st || desc->m == 0) return st;
   if (desc->n > 0 && !cache) return refuse(who, "a pointer is null");
   const void *ptrs[] = {indx, pntrb, pntre, q, cache, lambda, o, work};
   st = check_pointers(who, ptrs, 8);
   if (st) return st;
   p.cache = (const uint8_t *)cache;
   p.ldc = ldc;
   p.hdc = hdc;
   return launch_rows_kv4(p, dc, desc->maps, (hipStream_t)stream);
}

}  // extern "C"
