// paged.cuh - what the paged KV-cache kernels share: the cache description,
// the arguments of the attention kernels and the element types.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>

#include "common.cuh"

namespace ddq {

// One pool of pages: k and v [num_pages, Hkv, page, D] through element strides
// (D contiguous), pages of 2^page_shift rows.
struct PgCache {
  void* k;
  void* v;
  int64_t page_stride, head_stride, row_stride;
  int num_pages, page_shift;
  int Hkv, D;
  int* err;  // the device error word
};

__device__ __forceinline__ void pg_error(const PgCache& c, int code) { atomicCAS(c.err, 0, code); }

struct PgAttnArgs {
  PgCache c;
  const void* q;            // [T, Hq, D], element strides
  int64_t q_ts, q_hs;
  void* out;                // [T, Hq, D]
  int64_t o_ts, o_hs;
  const int* table;         // [R, width], row stride table_stride
  int64_t table_stride;
  int width;
  const int* lens;          // [R] keys of each request in its own pages
  const int* cu;            // [R + 1] first query row of each request; null: one row each
  const int* bidir;         // [R] or null: own keys every row of the request may attend
  const int* prefix_pages;  // shared prefix (its rows come before the own ones) or null
  int prefix_len;
  const float* slopes;      // [Hq] or null
  float scale, cap;
  int T, R, Hq;
  int G;                    // query heads of a key/value head
};

// tanh(y) = y P(y^2) for |y| <= 1/2: P the minimax polynomial of degree 4 of
// tanh(sqrt u) / sqrt(u) on [0, 1/4] (Remez, relative error 2^-26).
constexpr float PG_TANH0 = 0.999999987f, PG_TANH1 = -0.333330694f, PG_TANH2 = 0.133247793f,
                PG_TANH3 = -0.0529860753f, PG_TANH4 = 0.0171350066f;

// A capped score in log2 units, A tanh(y) with y = ratio v = kk v / A: by the
// polynomial up to |y| = 1/2 and, where `large`, as A - 2 A / (exp(2 y) + 1)
// above.  The latter alone is off by a few 2^-23 of the cap, which is not small
// against a score far below it (3 under a cap of 10^6 came out as 2.9).
__device__ __forceinline__ float pg_capped(float v, float kk, float ratio, float A, bool large) {
  const float y = v * ratio, w = y * y;
  const float p =
      fmaf(fmaf(fmaf(fmaf(PG_TANH4, w, PG_TANH3), w, PG_TANH2), w, PG_TANH1), w, PG_TANH0);
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y * 2.885390082f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 1.f));
  return large && !(fabsf(y) <= 0.5f) ? fmaf(-2.f * A, r, A) : v * kk * p;
}

// scale / cap, finite also under the smallest cap, so that a score of 0 stays 0
__device__ __forceinline__ float pg_cap_ratio(float scale, float cap) {
  return fminf(fmaxf(scale / cap, -3.4e38f), 3.4e38f);
}

// Parts of a split key axis: part z of row t * Hq + h holds the row's output
// over its keys, o[z][row][D], and log2 of the sum of its weights, lse[z][row]
// (-inf: no keys, o not written).  o null: one part, written to the output itself.
struct PgParts {
  float* o;
  float* lse;
  int64_t rows;
  int count;
};

template <typename T>
struct PgType;
template <>
struct PgType<__half> {
  static __device__ __forceinline__ float2 to_f2(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct PgType<__nv_bfloat16> {
  static __device__ __forceinline__ float2 to_f2(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// Keys of request r in its own pages: the length, never more than its table
// row holds (a longer one is an error of the caller's, recorded).
__device__ __forceinline__ int pg_clamp_len(const PgAttnArgs& a, int n) {
  const int64_t hold = (int64_t)a.width << a.c.page_shift;
  if (n <= hold) return n < 0 ? 0 : n;
  pg_error(a.c, DDQ_ERR_PAGE);
  return (int)hold;
}

__device__ __forceinline__ int pg_len(const PgAttnArgs& a, int r) {
  return pg_clamp_len(a, a.lens[r]);
}

// A page number as the tables hold it, -1 (recorded) for one outside the pool.
__device__ __forceinline__ int pg_check(const PgCache& c, int page) {
  if ((unsigned)page < (unsigned)c.num_pages) return page;
  pg_error(c, DDQ_ERR_PAGE);
  return -1;
}

constexpr int kPlanMaxR = 8192;  // requests of a plan
int launch_plan_step(const int* cached, const int* fresh, int* table, int64_t table_stride,
                     int width, const int* free_pages, int num_free, const int* free_head,
                     int page_shift, int64_t prefix_len, int* cu, int* lens, int64_t* slots,
                     int64_t* positions, int* seq_ids, int* free_head_out, int R, int T,
                     cudaStream_t s);
int launch_paged_rope_kv(const void* qkv, int64_t qkv_stride, const PgCache& c, bool bf16,
                         const float* cos, const float* sin, int64_t max_pos,
                         const int64_t* slots, const int64_t* positions, void* q_out, int64_t T,
                         int Hq, cudaStream_t s);
int tc_splits(int64_t T, int64_t R, int Hq, int Hkv, int64_t keys, bool ragged, int sms);
int launch_paged_tc(const PgAttnArgs& a, bool bf16, const PgParts& parts, int splits,
                    unsigned long long tmo, int debug_flags, cudaStream_t s);
int pg_tensor_map(CUtensorMap* m, const PgCache& c, const void* base, bool bf16, int rows);
// What a decode call runs and where its workspace holds what: the prefix parts
// and the own part (as PgParts), then the side slots.
struct DcPlan {
  int ctas, splits;
  size_t off_lse, off_so, off_sl, off_seg, bytes;
};
DcPlan dc_plan(int64_t B, int Hq, int Hkv, int D, int64_t keys, int64_t prefix, int sms);
int launch_paged_decode(const PgAttnArgs& a, bool bf16, void* ws, const DcPlan& plan,
                        unsigned long long tmo, int debug_flags, cudaStream_t s);
int launch_paged_merge(const PgAttnArgs& a, bool bf16, const PgParts& parts, cudaStream_t s);

}  // namespace ddq
