// C ABI of the paged key-value cache: argument checks (host only, before any HIP call) and launches.
#include <math.h>
#include <stdarg.h>

#include "ra_paged.h"

namespace ra {
int fail_with(int code, const char* fmt, va_list ap);
}

namespace {

using namespace ra;

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  fail_with(code, fmt, ap);
  va_end(ap);
  return code;
}
int done(hipError_t e, const char* what) { return e == hipSuccess ? RA_OK : fail(RA_ERR_HIP, "%s: %s", what, hipGetErrorString(e)); }
bool misaligned(const void* p, unsigned bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

constexpr int64_t kMost32 = 0x7fffffff;
constexpr int64_t kMaxTokens = 1 << 30;  // of a sequence: positions and what is added to them fit 32 bits

int check_type(int dtype) {
  return dtype == RA_DTYPE_BF16 || dtype == RA_DTYPE_F16 ? RA_OK : fail(RA_ERR_DTYPE, "pages hold bf16 or fp16 (got dtype %d)", dtype);
}
int check_page_size(int size, int& shift) {
  if (size < 16 || size > 65536 || (size & (size - 1))) return fail(RA_ERR_SHAPE, "page_size must be a power of two from 16 to 65536 (got %d)", size);
  shift = __builtin_ctz(size);
  return RA_OK;
}
int check_rows(int B, int H, int D) {
  if (B <= 0 || B > RA_MAX_PAGED_ROWS) return fail(RA_ERR_SHAPE, "1 to %d sequences per call (got %d)", RA_MAX_PAGED_ROWS, B);
  if (H <= 0 || H > 65535) return fail(RA_ERR_SHAPE, "1 to 65535 heads (got %d)", H);
  if (D < 32 || D > 128 || D % 32) return fail(RA_ERR_HEAD_DIM, "head dim %d unsupported (32, 64, 96 or 128)", D);
  return RA_OK;
}
int check_table(const ra_page_table* t, int B, PageTable& r) {
  if (!t || !t->ptr) return fail(RA_ERR_NULL, "the page table is NULL");
  if (misaligned(t->ptr, 4)) return fail(RA_ERR_ALIGN, "the page table is not aligned to its elements");
  if (int e = check_page_size(t->page_size, r.shift)) return e;
  if (t->width <= 0 || t->n_pages <= 0) return fail(RA_ERR_SHAPE, "width and n_pages must be positive (got %d, %d)", t->width, t->n_pages);
  if ((int64_t)t->width * t->page_size > kMaxTokens) return fail(RA_ERR_SHAPE, "a table of %d pages of %d tokens holds more than 2^30", t->width, t->page_size);
  if ((int64_t)t->width * B > kMost32) return fail(RA_ERR_SHAPE, "a table of %d x %d entries has 2^31 or more", B, t->width);
  if (t->stride_b < (B > 1 ? t->width : 0)) return fail(RA_ERR_SHAPE, "rows of the page table overlap (stride %lld)", (long long)t->stride_b);
  r.at = t->ptr;
  r.sb = t->stride_b;
  r.width = t->width;
  r.n_pages = t->n_pages;
  return RA_OK;
}
int check_pool(const char* name, const ra_pool* p, int H, int D, int page_size, PoolArg& r) {
  if (!p || !p->ptr) return fail(RA_ERR_NULL, "%s is NULL", name);
  if (misaligned(p->ptr, 16) || ((p->stride_page | p->stride_token | p->stride_head) & 7))
    return fail(RA_ERR_ALIGN, "%s must be 16-byte aligned, its strides multiples of 8 elements", name);
  if (p->stride_page < 0 || p->stride_token < 0 || p->stride_head < 0 || p->stride_token > kMost32 || p->stride_head > kMost32 ||
      (page_size - 1) * p->stride_token + (H - 1) * p->stride_head + D > kMost32)
    return fail(RA_ERR_SHAPE, "%s: offsets within a page must lie in [0, 2^31) elements", name);
  r.ptr = static_cast<const unsigned short*>(p->ptr);
  r.sp = p->stride_page;
  r.st = (int)p->stride_token;
  r.sh = (int)p->stride_head;
  return RA_OK;
}
int check_strides(const char* name, const void* p, int64_t s0, int64_t s1, int n1, int D) {
  if (!p) return fail(RA_ERR_NULL, "%s is NULL", name);
  if (misaligned(p, 16) || ((s0 | s1) & 7)) return fail(RA_ERR_ALIGN, "%s must be 16-byte aligned, its strides multiples of 8 elements", name);
  if (s0 < 0 || s1 < 0 || s1 > kMost32 || (n1 - 1) * s1 + D > kMost32) return fail(RA_ERR_SHAPE, "%s: strides out of range", name);
  return RA_OK;
}
int check_lengths(const int32_t* a, const int32_t* b) {
  if (!a || !b) return fail(RA_ERR_NULL, "the lengths are NULL");
  return misaligned(a, 4) || misaligned(b, 4) ? fail(RA_ERR_ALIGN, "the lengths are not aligned to their elements") : RA_OK;
}

int paged_args(const ra_paged_params* p, PagedArgs& a, PagedShape& shape) {
  if (!p) return fail(RA_ERR_NULL, "the parameters are NULL");
  if (int e = check_type(p->dtype)) return e;
  if (int e = check_rows(p->B, p->H, p->D)) return e;
  if (p->group <= 0 || (int64_t)p->H * p->group > 65535) return fail(RA_ERR_SHAPE, "1 to 65535 query heads (got %d x %d)", p->H, p->group);
  if (p->window < 0) return fail(RA_ERR_BIAS, "window must be positive, or 0 for none (got %d)", p->window);
  if (!isfinite(p->sm_scale * kLog2e)) return fail(RA_ERR_SHAPE, "sm_scale must be finite, times log2(e) too");
  if (int e = check_table(&p->table, p->B, a.table)) return e;
  if (int e = check_strides("q", p->q, p->q_stride_b, p->q_stride_h, p->H * p->group, p->D)) return e;
  if (int e = check_pool("k", &p->k, p->H, p->D, p->table.page_size, a.k)) return e;
  if (int e = check_pool("v", &p->v, p->H, p->D, p->table.page_size, a.v)) return e;
  if (int e = check_lengths(p->lengths, p->lengths)) return e;
  if (p->pages && (p->n_pages_read <= 0 || (int64_t)p->n_pages_read * p->table.page_size > kMaxTokens))
    return fail(RA_ERR_SHAPE, "the pages that are read must hold 1 to 2^30 tokens (got %d of %d)", p->n_pages_read, p->table.page_size);
  if (misaligned(p->pages, 4) || misaligned(p->slopes, 4)) return fail(RA_ERR_ALIGN, "pages and slopes must be aligned to their elements");
  a.q = static_cast<const unsigned short*>(p->q);
  a.q_sb = p->q_stride_b;
  a.q_sh = (int)p->q_stride_h;
  a.lengths = p->lengths;
  a.pages = p->pages;
  a.count = p->n_pages_read;
  a.B = p->B;
  a.H = p->H;
  a.G = p->group;
  a.tiles = (p->group + kPartRows - 1) / kPartRows;
  a.window = p->window;
  a.slopes = p->slopes;
  a.scale2 = p->sm_scale * kLog2e;
  // (a window begins inside a tile of 32 keys)
  int64_t keys = (int64_t)(p->pages ? p->n_pages_read : p->table.width) * p->table.page_size;
  if (!p->pages && p->window > 0 && p->window + 31ll < keys) keys = p->window + 31ll;
  const int64_t steps = (keys + kStepKeys - 1) / kStepKeys, most = steps * p->B * p->H * a.tiles;
  if (most > kMost32) return fail(RA_ERR_TOO_LARGE, "%lld steps of %d keys are too many for one call", (long long)most, kStepKeys);
  shape = paged_shape(keys, (int64_t)p->B * p->H * a.tiles, p->D);
  return RA_OK;
}

}  // namespace

extern "C" {

int ra_page_slots(const ra_page_table* table, const int32_t* lengths, const int32_t* new_lengths, int32_t B, int32_t* free_pages,
                  const int32_t* free_state, int64_t* slots, int32_t n_slots, int32_t* starts, int32_t* granted, int32_t* free_state_out,
                  void* stream) {
  PageTable t;
  if (int e = check_rows(B, 1, 32)) return e;
  if (int e = check_table(table, B, t)) return e;
  if (int e = check_lengths(lengths, new_lengths)) return e;
  if (!free_pages || !free_state || !starts || !granted || !free_state_out || (n_slots > 0 && !slots)) return fail(RA_ERR_NULL, "an array is NULL");
  if (n_slots < 0) return fail(RA_ERR_SHAPE, "n_slots must not be negative (got %d)", n_slots);
  if (misaligned(free_pages, 4) || misaligned(free_state, 4) || misaligned(slots, 8) || misaligned(starts, 4) || misaligned(granted, 4) ||
      misaligned(free_state_out, 4))
    return fail(RA_ERR_ALIGN, "arrays must be aligned to their elements");
  const SlotsArgs a{table->ptr, t.sb, t.width, B, t.shift, lengths, new_lengths, free_pages, t.n_pages, free_state, (long long*)slots, n_slots, starts,
                    granted, free_state_out};
  return done(launch_slots(a, static_cast<hipStream_t>(stream)), "ra_page_slots");
}

int ra_write_pages(const void* k, int64_t k_stride_token, int64_t k_stride_head, const void* v, int64_t v_stride_token, int64_t v_stride_head,
                   int32_t src_dtype, int32_t T, int32_t H, int32_t D, const ra_pool* k_pool, const ra_pool* v_pool, int32_t dtype,
                   int32_t n_pages, int32_t page_size, const int64_t* slots, void* stream) {
  WriteArgs a;
  if (int e = check_type(dtype)) return e;
  if (src_dtype != RA_DTYPE_BF16 && src_dtype != RA_DTYPE_F16 && src_dtype != RA_DTYPE_F32)
    return fail(RA_ERR_DTYPE, "unknown source dtype %d", src_dtype);
  if (int e = check_rows(1, H, D)) return e;
  if (int e = check_page_size(page_size, a.shift)) return e;
  if (T < 0 || n_pages <= 0) return fail(RA_ERR_SHAPE, "n_pages must be positive and T not negative (got %d, %d)", n_pages, T);
  if (T == 0) return RA_OK;
  if ((int64_t)T * H * (D / 8) > kMost32) return fail(RA_ERR_TOO_LARGE, "%d tokens of %d x %d elements are too many for one call", T, H, D);
  if (int e = check_strides("k", k, k_stride_token, k_stride_head, H, D)) return e;
  if (int e = check_strides("v", v, v_stride_token, v_stride_head, H, D)) return e;
  if (int e = check_pool("k_pool", k_pool, H, D, page_size, a.k_pool)) return e;
  if (int e = check_pool("v_pool", v_pool, H, D, page_size, a.v_pool)) return e;
  if (!slots) return fail(RA_ERR_NULL, "slots is NULL");
  if (misaligned(slots, 8)) return fail(RA_ERR_ALIGN, "slots must be aligned to its elements");
  a.k = k;
  a.v = v;
  a.k_st = k_stride_token;
  a.k_sh = k_stride_head;
  a.v_st = v_stride_token;
  a.v_sh = v_stride_head;
  a.slots = (const long long*)slots;
  a.T = T;
  a.H = H;
  a.D = D;
  a.n_slots = (int64_t)n_pages * page_size;
  return done(launch_write(a, src_dtype, dtype, static_cast<hipStream_t>(stream)), "ra_write_pages");
}

int ra_page_means(const ra_pool* k_pool, int32_t dtype, const ra_page_table* table, const int32_t* lengths, const int32_t* new_lengths, int32_t B,
                  int32_t H, int32_t D, void* means, int64_t means_stride_page, int64_t means_stride_head, void* stream) {
  MeansArgs a;
  if (int e = check_type(dtype)) return e;
  if (int e = check_rows(B, H, D)) return e;
  if (int e = check_table(table, B, a.table)) return e;
  if (int e = check_pool("k_pool", k_pool, H, D, table->page_size, a.k)) return e;
  if (int e = check_lengths(lengths, new_lengths)) return e;
  if (int e = check_strides("means", means, means_stride_page, means_stride_head, H, D)) return e;
  a.before = lengths;
  a.after = new_lengths;
  a.means = static_cast<unsigned short*>(means);
  a.means_sp = means_stride_page;
  a.means_sh = (int)means_stride_head;
  a.B = B;
  a.H = H;
  a.D = D;
  return done(launch_means(a, dtype, static_cast<hipStream_t>(stream)), "ra_page_means");
}

int64_t ra_select_pages_workspace(const ra_page_table* table, int32_t B, int32_t H) {
  return table && table->width > 0 && B > 0 && H > 0 ? select_workspace(table->width, (int64_t)B * H) : 0;
}
int ra_select_pages(const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* means, int64_t means_stride_page, int64_t means_stride_head,
                    int32_t dtype, const ra_page_table* table, const int32_t* lengths, int32_t B, int32_t H, int32_t group, int32_t D, int32_t count,
                    int32_t first, int32_t last, int32_t* pages, void* workspace, int64_t workspace_bytes, void* stream) {
  SelectArgs a;
  if (int e = check_type(dtype)) return e;
  if (int e = check_rows(B, H, D)) return e;
  if (group <= 0 || (int64_t)H * group > 65535) return fail(RA_ERR_SHAPE, "1 to 65535 query heads (got %d x %d)", H, group);
  if (int e = check_table(table, B, a.table)) return e;
  if (count <= 0 || (int64_t)count * table->page_size > kMaxTokens || first < 0 || last < 0 || (int64_t)first + last > count)
    return fail(RA_ERR_SHAPE, "count must be positive, its tokens at most 2^30, and hold the first and last pages (got %d, %d, %d)", count, first, last);
  if ((int64_t)B * H * count > kMost32) return fail(RA_ERR_TOO_LARGE, "%d x %d x %d pages are too many for one call", B, H, count);
  if (int e = check_strides("q", q, q_stride_b, q_stride_h, H * group, D)) return e;
  if (int e = check_strides("means", means, means_stride_page, means_stride_head, H, D)) return e;
  if (int e = check_lengths(lengths, lengths)) return e;
  if (!pages) return fail(RA_ERR_NULL, "pages is NULL");
  if (misaligned(pages, 4)) return fail(RA_ERR_ALIGN, "pages must be aligned to its elements");
  const int64_t need = ra_select_pages_workspace(table, B, H);
  if (table->width > count && need > 0) {
    if (!workspace || workspace_bytes < need) return fail(RA_ERR_NULL, "a workspace of %lld bytes is needed", (long long)need);
    if (misaligned(workspace, 16)) return fail(RA_ERR_ALIGN, "the workspace must be 16-byte aligned");
  }
  a.q = static_cast<const unsigned short*>(q);
  a.q_sb = q_stride_b;
  a.q_sh = (int)q_stride_h;
  a.means = static_cast<const unsigned short*>(means);
  a.means_sp = means_stride_page;
  a.means_sh = (int)means_stride_head;
  a.lengths = lengths;
  a.B = B;
  a.H = H;
  a.G = group;
  a.D = D;
  a.count = count;
  a.first = first;
  a.last = last;
  a.keys = static_cast<unsigned long long*>(workspace);
  a.pages = pages;
  return done(launch_select(a, dtype, static_cast<hipStream_t>(stream)), "ra_select_pages");
}

int64_t ra_paged_attention_workspace(const ra_paged_params* p) {
  PagedArgs a;
  PagedShape shape;
  return paged_args(p, a, shape) == RA_OK ? shape.workspace : 0;  // (the call itself says what is wrong)
}
int ra_paged_attention(const ra_paged_params* p, void* out, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  PagedArgs a;
  PagedShape shape;
  if (int e = paged_args(p, a, shape)) return e;
  if (!out || !lse) return fail(RA_ERR_NULL, "out or lse is NULL");
  if (misaligned(out, 16) || misaligned(lse, 4)) return fail(RA_ERR_ALIGN, "out must be 16-byte aligned, lse to its elements");
  if (shape.workspace > 0) {
    if (!workspace || workspace_bytes < shape.workspace) return fail(RA_ERR_NULL, "a workspace of %lld bytes is needed", shape.workspace);
    if (misaligned(workspace, 16)) return fail(RA_ERR_ALIGN, "the workspace must be 16-byte aligned");
  }
  a.out = static_cast<unsigned short*>(out);
  a.lse = lse;
  return done(launch_paged(a, p->D, p->dtype, shape, workspace, static_cast<hipStream_t>(stream)), "ra_paged_attention");
}
int ra_put_floats(const float* values, int32_t n, float* to, void* stream) {
  if (n < 0 || n > 65535) return fail(RA_ERR_SHAPE, "0 to 65535 numbers, as many as there are query heads (got %d)", n);
  if (n == 0) return RA_OK;
  if (!values || !to) return fail(RA_ERR_NULL, "an array is NULL");
  if (misaligned(values, 4) || misaligned(to, 4)) return fail(RA_ERR_ALIGN, "arrays must be aligned to their elements");
  return done(launch_put(values, n, to, static_cast<hipStream_t>(stream)), "ra_put_floats");
}

}  // extern "C"
