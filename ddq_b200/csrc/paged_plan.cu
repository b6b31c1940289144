// paged_plan.cu - the step plan of a paged KV cache: which new pages each
// request takes, and for every new token its slot, position and request.
//
//   lens_r  = cached_r + new_r
//   have_r  = ceil(cached_r / page)            pages the request holds already
//   need_r  = ceil(lens_r / page) - have_r     pages it takes now
//   first_r = free_head + sum_{r' < r} need_r'
//   table[r, have_r + i] = free_pages[first_r + i],  i < need_r
//   cu_r    = sum_{r' < r} new_r'
//   token t of request r (cu_r <= t < cu_{r+1}), i = t - cu_r, p = cached_r + i:
//     slot = table[r, p / page] * page + p % page,  position = prefix_len + p
//
// One launch.  Both sums run over all requests, and a step has few of them
// (at most kPlanMaxR), so every CTA makes the whole scan itself in shared memory
// (8 bytes a request, from L2 after the first CTA) instead of waiting for the
// other CTAs' parts.  A token or a fresh page then finds its request by binary
// search, so one long prompt among many short ones is spread over all threads;
// a token of a fresh page reads the free list, not the table row that another
// CTA may be writing.  Latency bound at the sizes of a step.
#include "launch.cuh"
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace ddq {

constexpr int PL_NT = 512;

struct PlArgs {
  const int* cached;
  const int* fresh;
  int* table;
  int64_t table_stride;
  int width;
  const int* free_pages;
  int num_free;
  const int* free_head;
  int page_shift;
  int64_t prefix_len;
  int* cu;
  int* lens;
  int64_t* slots;
  int64_t* positions;
  int* seq_ids;
  int* free_head_out;
  int R, T;
};

// Lengths outside [0, PL_MAXLEN] are taken as its ends, so that no length on
// the device, however wrong, leads to an index outside the arrays.
constexpr int PL_MAXLEN = 0x7fffff00;

__device__ __forceinline__ int pl_cached(const PlArgs& a, int r) {
  return min(max(a.cached[r], 0), PL_MAXLEN);
}

__device__ __forceinline__ int pl_pages(int n, int shift) {
  return (int)(((int64_t)n + (1 << shift) - 1) >> shift);
}

// largest r < R with base[r] <= x (base ascending, base[0] = 0 <= x)
__device__ __forceinline__ int pl_find(const int* base, int R, int x) {
  int lo = 0, hi = R;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (base[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(PL_NT) plan_step_kernel(const PlArgs a) {
  extern __shared__ int pl_smem[];
  int* cu = pl_smem;                  // [R + 1]
  int* first = pl_smem + a.R + 1;     // [R + 1], without the head
  __shared__ int wsum[2][PL_NT / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int head = a.free_head ? *a.free_head : 0;

  // exclusive sums of new tokens and of pages, PL_NT requests at a time
  int run0 = 0, run1 = 0;
  for (int base = 0; base < a.R; base += PL_NT) {
    const int r = base + threadIdx.x;
    int n = 0, need = 0;
    if (r < a.R) {
      const int c = pl_cached(a, r);
      n = min(max(a.fresh[r], 0), PL_MAXLEN - c);
      need = pl_pages(c + n, a.page_shift) - pl_pages(c, a.page_shift);
      if (blockIdx.x == 0) a.lens[r] = c + n;
    }
    int s0 = n, s1 = need;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u0 = __shfl_up_sync(0xffffffffu, s0, o), u1 = __shfl_up_sync(0xffffffffu, s1, o);
      if (lane >= o) {
        s0 += u0;
        s1 += u1;
      }
    }
    if (lane == 31) {
      wsum[0][warp] = s0;
      wsum[1][warp] = s1;
    }
    __syncthreads();
    int b0 = run0, b1 = run1;
    for (int w = 0; w < PL_NT / 32; ++w) {
      const int x0 = wsum[0][w], x1 = wsum[1][w];
      if (w < warp) {
        b0 += x0;
        b1 += x1;
      }
      run0 += x0;
      run1 += x1;
    }
    if (r < a.R) {
      cu[r] = b0 + s0 - n;
      first[r] = b1 + s1 - need;
      if (blockIdx.x == 0) a.cu[r] = cu[r];
    }
    __syncthreads();  // wsum is free again; the last pass publishes cu and first
  }
  const int total = run0, pages = run1;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.cu[a.R] = total;
    *a.free_head_out = head + pages;
  }
  auto fresh_page = [&](int i) {  // i-th page handed out by this step
    const int64_t k = (int64_t)head + i;
    const int pg = k >= 0 && k < a.num_free ? a.free_pages[k] : -1;
    return pg < 0 ? -1 : pg;
  };
  const int stride = gridDim.x * PL_NT, t0 = blockIdx.x * PL_NT + threadIdx.x;
  for (int t = t0; t < a.T; t += stride) {
    int64_t slot = -1, pos = 0;
    int seq = -1;
    if (t < total) {
      seq = pl_find(cu, a.R, t);
      const int c = pl_cached(a, seq), p = c + (t - cu[seq]);
      const int col = p >> a.page_shift, have = pl_pages(c, a.page_shift);
      int pg = -1;
      if ((unsigned)col < (unsigned)a.width)
        pg = col < have ? a.table[(size_t)seq * a.table_stride + col]
                        : fresh_page(first[seq] + col - have);
      if (pg >= 0) slot = ((int64_t)pg << a.page_shift) + (p & ((1 << a.page_shift) - 1));
      pos = a.prefix_len + p;
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
    a.seq_ids[t] = seq;
  }
  for (int i = t0; i < pages; i += stride) {
    const int r = pl_find(first, a.R, i);
    const int col = pl_pages(pl_cached(a, r), a.page_shift) + (i - first[r]);
    if ((unsigned)col < (unsigned)a.width) a.table[(size_t)r * a.table_stride + col] = fresh_page(i);
  }
}

int launch_plan_step(const int* cached, const int* fresh, int* table, int64_t table_stride,
                     int width, const int* free_pages, int num_free, const int* free_head,
                     int page_shift, int64_t prefix_len, int* cu, int* lens, int64_t* slots,
                     int64_t* positions, int* seq_ids, int* free_head_out, int R, int T,
                     cudaStream_t s) {
  const int sms = device_sm_count(current_device());
  if (sms <= 0) return DDQ_ERR_DEVICE;
  PlArgs a{cached, fresh, table, table_stride, width, free_pages, num_free, free_head,
           page_shift, prefix_len, cu, lens, slots, positions, seq_ids, free_head_out, R, T};
  int64_t blocks = ((int64_t)T + PL_NT - 1) / PL_NT;
  blocks = blocks < 1 ? 1 : blocks > sms ? sms : blocks;
  const int smem = 2 * (R + 1) * (int)sizeof(int);
  static SmemAttrOnce attr;
  const int st = ensure_smem_attr(attr, current_device(), plan_step_kernel,
                                  2 * (kPlanMaxR + 1) * (int)sizeof(int));
  if (st) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(PL_NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, plan_step_kernel, a) != cudaSuccess) {
    cudaGetLastError();
    return DDQ_ERR_LAUNCH;
  }
  return check_launch();
}

}  // namespace ddq
