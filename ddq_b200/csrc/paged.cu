// paged.cu - the extern "C" entry points of the paged KV-cache operators
// (include/ddq_b200.h): argument validation and the hand-over to the kernels.
#include <cmath>

#include "launch.cuh"
#include "paged.cuh"

namespace ddq {
namespace {

constexpr int64_t kIntMax = 0x7fffffff;

int page_shift_of(int64_t page_size) {
  for (int sh = 0; (int64_t)1 << sh <= DDQ_PAGE_SIZE_MAX; ++sh)
    if (page_size == (int64_t)1 << sh) return page_size >= DDQ_PAGE_SIZE_MIN ? sh : -1;
  return -1;
}

int check_cache(const ddq_paged_cache* c, PgCache* out) {
  if (!c || !c->k || !c->v) return DDQ_ERR_INVALID_ARGUMENT;
  if (c->dtype != DDQ_DTYPE_F16 && c->dtype != DDQ_DTYPE_BF16) return DDQ_ERR_INVALID_ARGUMENT;
  const int sh = page_shift_of(c->page_size);
  if (sh < 0 || (c->D != 64 && c->D != 128) || c->Hkv < 1 || c->Hkv > 1024 || c->num_pages < 1 ||
      c->num_pages > kIntMax)
    return DDQ_ERR_SHAPE;
  if (c->page_stride < 0 || c->head_stride < 0 || c->row_stride < c->D) return DDQ_ERR_SHAPE;
  if (!aligned16(c->k) || !aligned16(c->v) || c->page_stride % 8 != 0 ||
      c->head_stride % 8 != 0 || c->row_stride % 8 != 0)
    return DDQ_ERR_ALIGNMENT;
  *out = PgCache{c->k, c->v, c->page_stride, c->head_stride, c->row_stride,
                 (int)c->num_pages, sh, (int)c->Hkv, (int)c->D, nullptr};
  return DDQ_OK;
}

// A written tensor: no element at two index tuples (dims of n[i] elements at
// strides st[i], above a contiguous run of `inner`).
bool distinct(int64_t inner, const int64_t* n, const int64_t* st, int dims) {
  int order[3];
  for (int i = 0; i < dims; ++i) {
    int j = i;
    for (; j > 0 && st[order[j - 1]] > st[i]; --j) order[j] = order[j - 1];
    order[j] = i;
  }
  int64_t extent = inner;
  for (int i = 0; i < dims; ++i) {
    const int k = order[i];
    if (n[k] <= 1) continue;
    if (st[k] < extent) return false;
    extent = (n[k] - 1) * st[k] + extent;
  }
  return true;
}

// Index arrays (null: absent) on their natural alignment.
template <typename... P>
bool aligned_as(const P*... p) {
  return ((reinterpret_cast<uintptr_t>(p) % alignof(P) == 0) && ...);
}

int check_attn(const void* q, int64_t q_ts, int64_t q_hs, const void* out, int64_t o_ts,
               int64_t o_hs, const int* table, int64_t table_stride, int64_t table_width,
               const int* lens, const int* prefix_pages, const float* slopes, int64_t prefix_len,
               float scale, float softcap, int64_t T, int64_t Hq, const PgCache& c) {
  if (!q || !out || !table || !lens) return DDQ_ERR_INVALID_ARGUMENT;
  if (!std::isfinite(scale) || !std::isfinite(softcap) || softcap < 0.f)
    return DDQ_ERR_INVALID_ARGUMENT;
  if (T > kIntMax || Hq < 1 || Hq > 1024 || Hq % c.Hkv != 0 || T * Hq > kIntMax || table_width < 1 ||
      table_width > kIntMax || table_stride < table_width || q_ts < 0 || o_ts < 0 || q_hs < 0 ||
      o_hs < 0)
    return DDQ_ERR_SHAPE;
  // positions are 32-bit, up to a tile behind the last
  if (prefix_len + (table_width << c.page_shift) > kIntMax - 255) return DDQ_ERR_SHAPE;
  const int64_t n[2] = {T, Hq}, st[2] = {o_ts, o_hs};
  if (!distinct(c.D, n, st, 2)) return DDQ_ERR_SHAPE;
  if (!aligned16(q) || !aligned16(out) || q_ts % 8 != 0 || q_hs % 8 != 0 || o_ts % 8 != 0 ||
      o_hs % 8 != 0 || !aligned_as(table, lens, prefix_pages, slopes))
    return DDQ_ERR_ALIGNMENT;
  return DDQ_OK;
}

// A run of memory, and whether two of them, or one and a row of a table, share a byte.
struct Span {
  const void* p;
  int64_t bytes;
};

bool meet(const Span& a, const Span& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
  return a.bytes > 0 && b.bytes > 0 && x < y + b.bytes && y < x + a.bytes;
}

bool meets_row(const Span& a, const int32_t* table, int64_t stride, int64_t width, int64_t rows) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), t = reinterpret_cast<uintptr_t>(table);
  const uintptr_t end = t + 4 * (uintptr_t)width;  // of the first row
  // the first row that ends behind the start of a
  const uintptr_t r = x < end ? 0 : (x - end) / (4 * (uintptr_t)stride) + 1;
  return a.bytes > 0 && r < (uintptr_t)rows && t + r * 4 * (uintptr_t)stride < x + a.bytes;
}

}  // namespace
}  // namespace ddq

using namespace ddq;

extern "C" int ddq_plan_step(const int32_t* cached, const int32_t* new_tokens,
                             int32_t* block_table, int64_t table_stride, int64_t table_width,
                             const int32_t* free_pages, int64_t num_free,
                             const int32_t* free_head, int64_t page_size, int64_t prefix_len,
                             int32_t* cu_new, int32_t* lens, int64_t* slots, int64_t* positions,
                             int32_t* seq_ids, int32_t* free_head_out, int64_t R, int64_t T,
                             void* stream) {
  if (R < 1 || R > kPlanMaxR || T < 0 || table_width < 1 || table_stride < table_width ||
      num_free < 0 || prefix_len < 0 || T > kIntMax || table_width > kIntMax || num_free > kIntMax ||
      page_shift_of(page_size) < 0)
    return DDQ_ERR_SHAPE;
  if (!cached || !new_tokens || !block_table || (num_free > 0 && !free_pages) || !cu_new ||
      !lens || (T > 0 && (!slots || !positions || !seq_ids)) || !free_head_out)
    return DDQ_ERR_INVALID_ARGUMENT;
  // every CTA reads all of the inputs while others write: what is written lies apart
  const Span mem[] = {{cu_new, 4 * (R + 1)}, {lens, 4 * R},      {slots, 8 * T},
                      {positions, 8 * T},    {seq_ids, 4 * T},   {free_head_out, 4},
                      {cached, 4 * R},       {new_tokens, 4 * R}, {free_pages, 4 * num_free},
                      {free_head, free_head ? 4 : 0}};
  constexpr int kWritten = 6;
  for (int i = 0; i < (int)(sizeof(mem) / sizeof(mem[0])); ++i) {
    if (meets_row(mem[i], block_table, table_stride, table_width, R))
      return DDQ_ERR_INVALID_ARGUMENT;
    for (int j = 0; j < i && j < kWritten; ++j)
      if (meet(mem[i], mem[j])) return DDQ_ERR_INVALID_ARGUMENT;
  }
  if (!aligned_as(cached, new_tokens, block_table, free_pages, free_head, cu_new, lens, slots,
                  positions, seq_ids, free_head_out))
    return DDQ_ERR_ALIGNMENT;
  return launch_plan_step(cached, new_tokens, block_table, table_stride, (int)table_width,
                          free_pages, (int)num_free, free_head, page_shift_of(page_size),
                          prefix_len, cu_new, lens, slots, positions, seq_ids, free_head_out,
                          (int)R, (int)T, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int ddq_paged_rope_kv(const void* qkv, int64_t qkv_stride,
                                 const ddq_paged_cache* cache, const float* cos, const float* sin,
                                 int64_t max_pos, const int64_t* slots, const int64_t* positions,
                                 void* q_out, int64_t T, int64_t Hq, void* stream) {
  if (T < 0 || max_pos < 0 || Hq < 1 || Hq > 1024) return DDQ_ERR_SHAPE;
  PgCache c;
  const int st = check_cache(cache, &c);
  if (st) return st;
  if (T == 0) return DDQ_OK;
  if (!qkv || !cos || !sin || !slots || !positions || !q_out) return DDQ_ERR_INVALID_ARGUMENT;
  const int64_t n[3] = {c.num_pages, c.Hkv, (int64_t)1 << c.page_shift};
  const int64_t pst[3] = {c.page_stride, c.head_stride, c.row_stride};
  if (!distinct(c.D, n, pst, 3)) return DDQ_ERR_SHAPE;
  if (T > kIntMax || qkv_stride < (Hq + 2 * c.Hkv) * c.D) return DDQ_ERR_SHAPE;
  if (!aligned16(qkv) || qkv_stride % 8 != 0 || !aligned16(cos) || !aligned16(sin) ||
      !aligned16(q_out) || !aligned_as(slots, positions))
    return DDQ_ERR_ALIGNMENT;
  return launch_paged_rope_kv(qkv, qkv_stride, c, cache->dtype == DDQ_DTYPE_BF16, cos, sin,
                              max_pos, slots, positions, q_out, T, (int)Hq,
                              reinterpret_cast<cudaStream_t>(stream));
}

namespace {
int sm_count() {
  const int n = device_sm_count(current_device());
  return n > 0 ? n : 148;
}
// o [count][rows][D] and lse [count][rows], fp32
size_t parts_bytes(int64_t rows, int64_t D, int count) {
  return count > 1 ? (size_t)count * rows * (D + 1) * sizeof(float) : 0;
}
PgParts make_parts(void* ws, int64_t rows, int64_t D, int count) {
  if (count <= 1) return PgParts{nullptr, nullptr, rows, 1};
  float* o = static_cast<float*>(ws);
  return PgParts{o, o + (size_t)count * rows * D, rows, count};
}
bool attn_shape(int64_t T, int64_t R, int64_t Hq, int64_t Hkv, int64_t D, int64_t table_width,
                int64_t page_size, int64_t prefix_len) {
  return T > 0 && R > 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && D > 0 && table_width > 0 &&
         page_size > 0 && prefix_len >= 0;
}
}  // namespace

extern "C" size_t ddq_paged_prefill_attention_workspace_size(int64_t T, int64_t R, int64_t Hq,
                                                             int64_t Hkv, int64_t D,
                                                             int64_t table_width,
                                                             int64_t page_size,
                                                             int64_t prefix_len) {
  if (!attn_shape(T, R, Hq, Hkv, D, table_width, page_size, prefix_len)) return 0;
  const int s = tc_splits(T, R, (int)Hq, (int)Hkv, prefix_len + table_width * page_size, true,
                          sm_count());
  return parts_bytes(T * Hq, D, s);
}

extern "C" size_t ddq_paged_decode_attention_workspace_size(int64_t B, int64_t Hq, int64_t Hkv,
                                                            int64_t D, int64_t table_width,
                                                            int64_t page_size,
                                                            int64_t prefix_len) {
  if (!attn_shape(B, B, Hq, Hkv, D, table_width, page_size, prefix_len)) return 0;
  return dc_plan(B, (int)Hq, (int)Hkv, (int)D, table_width * page_size, prefix_len, sm_count())
      .bytes;
}

extern "C" int ddq_paged_prefill_attention(
    const void* q, int64_t q_token_stride, int64_t q_head_stride, const ddq_paged_cache* cache,
    const int32_t* block_table, int64_t table_stride, int64_t table_width, const int32_t* cu_new,
    const int32_t* lens, const int32_t* bidir, const int32_t* prefix_pages, int64_t prefix_len,
    const float* slopes, float scale, float softcap, void* out, int64_t out_token_stride,
    int64_t out_head_stride, int64_t T, int64_t R, int64_t Hq, void* workspace,
    size_t workspace_bytes, void* stream) {
  if (T < 0 || R < 0 || R > kIntMax || prefix_len < 0 || prefix_len > kIntMax / 2)
    return DDQ_ERR_SHAPE;
  PgCache c;
  int st = check_cache(cache, &c);
  if (st) return st;
  if (T == 0 || R == 0) return DDQ_OK;
  if (!cu_new || (prefix_len > 0 && !prefix_pages)) return DDQ_ERR_INVALID_ARGUMENT;
  st = check_attn(q, q_token_stride, q_head_stride, out, out_token_stride, out_head_stride,
                  block_table, table_stride, table_width, lens, prefix_pages, slopes, prefix_len,
                  scale, softcap, T, Hq, c);
  if (st) return st;
  if (!aligned_as(cu_new, bidir)) return DDQ_ERR_ALIGNMENT;
  if (!(c.err = device_error_word())) return DDQ_ERR_DEVICE;
  const bool bf16 = cache->dtype == DDQ_DTYPE_BF16;
  const int splits = tc_splits(T, R, (int)Hq, c.Hkv,
                               prefix_len + (table_width << c.page_shift), true, sm_count());
  if (splits > 1 && (!workspace || workspace_bytes < parts_bytes(T * Hq, c.D, splits)))
    return DDQ_ERR_WORKSPACE;
  if (splits > 1 && !aligned16(workspace)) return DDQ_ERR_ALIGNMENT;
  const PgParts parts = make_parts(workspace, T * Hq, c.D, splits);
  PgAttnArgs a{c, q, q_token_stride, q_head_stride, out, out_token_stride, out_head_stride,
               block_table, table_stride, (int)table_width, lens, cu_new, bidir, prefix_pages,
               (int)prefix_len, slopes, scale, softcap, (int)T, (int)R, (int)Hq, (int)Hq / c.Hkv};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  st = launch_paged_tc(a, bf16, parts, splits, wait_timeout_ns(), debug_flags(), s);
  if (st || splits == 1) return st;
  return launch_paged_merge(a, bf16, parts, s);
}

extern "C" int ddq_paged_decode_attention(
    const void* q, int64_t q_token_stride, int64_t q_head_stride, const ddq_paged_cache* cache,
    const int32_t* block_table, int64_t table_stride, int64_t table_width, const int32_t* lens,
    const int32_t* prefix_pages, int64_t prefix_len, const float* slopes, float scale,
    float softcap, void* out, int64_t out_token_stride, int64_t out_head_stride, int64_t B,
    int64_t Hq, void* workspace, size_t workspace_bytes, void* stream) {
  if (B < 0 || prefix_len < 0 || prefix_len > kIntMax / 2) return DDQ_ERR_SHAPE;
  PgCache c;
  int st = check_cache(cache, &c);
  if (st) return st;
  if (B == 0) return DDQ_OK;
  if (prefix_len > 0 && !prefix_pages) return DDQ_ERR_INVALID_ARGUMENT;
  st = check_attn(q, q_token_stride, q_head_stride, out, out_token_stride, out_head_stride,
                  block_table, table_stride, table_width, lens, prefix_pages, slopes, prefix_len,
                  scale, softcap, B, Hq, c);
  if (st) return st;
  const DcPlan plan = dc_plan(B, (int)Hq, c.Hkv, c.D, table_width << c.page_shift, prefix_len,
                              sm_count());
  if (!workspace || workspace_bytes < plan.bytes) return DDQ_ERR_WORKSPACE;
  if (!aligned16(workspace)) return DDQ_ERR_ALIGNMENT;
  if (!(c.err = device_error_word())) return DDQ_ERR_DEVICE;
  PgAttnArgs a{c, q, q_token_stride, q_head_stride, out, out_token_stride, out_head_stride,
               block_table, table_stride, (int)table_width, lens, nullptr, nullptr, prefix_pages,
               (int)prefix_len, slopes, scale, softcap, (int)B, (int)B, (int)Hq, (int)Hq / c.Hkv};
  return launch_paged_decode(a, cache->dtype == DDQ_DTYPE_BF16, workspace, plan,
                             wait_timeout_ns(), debug_flags(), reinterpret_cast<cudaStream_t>(stream));
}
