// paged_attn.cu - attention over the pages of a paged KV cache: the new tokens
// of ragged requests (prompts, chunks of prompts) and single decode tokens
// behind a shared prefix.
//
// Row (t, h), key head g = h / (Hq / Hkv), at position p, attends the keys j of
// its own request (and of the shared prefix, which comes first) with j < end:
//   s_j = scale q . k_j          (capped: cap * tanh(s_j / cap))
//   z_j = s_j - slope_h |p - j|
//   o   = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m),   m = max_j z_j
// and o = 0 where there is no such key.  A prompt's row has
// end = max(p + 1, prefix_len + min(bidir, len)), a decode row all keys.
//
// One warp per row: lane = D / 32 dimensions, one key at a time, an online
// softmax in fp32.  Bound by the shuffles of the dot product.
#include "launch.cuh"
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace ddq {

template <typename E, int D>
__global__ void __launch_bounds__(256) paged_attention_row_kernel(const PgAttnArgs a) {
  using Ty = PgType<E>;
  constexpr int DPL = D / 32;
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= (int64_t)a.T * a.Hq) return;
  const int t = (int)(row / a.Hq), h = (int)(row % a.Hq), g = h / (a.Hq / a.c.Hkv);
  int r = t, n = 1, i = 0;
  if (a.cu) {  // the request of the row; rows behind the last request stay as they are
    int lo = 0, hi = a.R;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu[mid] <= t) lo = mid; else hi = mid;
    }
    r = lo;
    const int c0 = a.cu[r], c1 = a.cu[r + 1];
    if (t < c0 || t >= c1) return;
    n = c1 - c0;
    i = t - c0;
  }
  const int len = pg_len(a, r);
  const int pos = a.prefix_len + len - n + i;
  int end = a.prefix_len + len;
  if (a.cu) {
    end = pos + 1;
    if (a.bidir) end = max(end, a.prefix_len + min(a.bidir[r], len));
  }
  float q[DPL], o[DPL], m = -INFINITY, l = 0.f;
  const E* qr = reinterpret_cast<const E*>(a.q) + t * a.q_ts + h * a.q_hs + lane * DPL;
#pragma unroll
  for (int e = 0; e < DPL; ++e) {
    q[e] = Ty::to_f(qr[e]);
    o[e] = 0.f;
  }
  const float slope = a.slopes ? a.slopes[h] : 0.f;
  const int ps = 1 << a.c.page_shift;
  for (int j = 0; j < end; ++j) {
    const bool shared = j < a.prefix_len;
    const int own = shared ? j : j - a.prefix_len;
    const int page = pg_check(a.c, shared ? a.prefix_pages[own >> a.c.page_shift]
                                          : a.table[r * a.table_stride + (own >> a.c.page_shift)]);
    if (page < 0) continue;
    const int64_t off = page * a.c.page_stride + g * a.c.head_stride +
                        (own & (ps - 1)) * a.c.row_stride + lane * DPL;
    const E* kr = reinterpret_cast<const E*>(a.c.k) + off;
    const E* vr = reinterpret_cast<const E*>(a.c.v) + off;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < DPL; ++e) s = fmaf(q[e], Ty::to_f(kr[e]), s);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= a.scale;
    if (a.cap > 0.f) s = a.cap * tanhf(s / a.cap);
    s -= slope * fabsf((float)(pos - j));
    const float mn = fmaxf(m, s);
    const float corr = __expf(m - mn), p = __expf(s - mn);
    l = l * corr + p;
#pragma unroll
    for (int e = 0; e < DPL; ++e) o[e] = fmaf(p, Ty::to_f(vr[e]), o[e] * corr);
    m = mn;
  }
  E* dst = reinterpret_cast<E*>(a.out) + t * a.o_ts + h * a.o_hs + lane * DPL;
#pragma unroll
  for (int e = 0; e < DPL; ++e) dst[e] = Ty::from_f(l > 0.f ? o[e] / l : (l == 0.f ? 0.f : l));
}

// Joins the parts of every row: o = sum_z 2^(lse_z - max) o_z / sum_z 2^(lse_z -
// max), in part order.  One warp per row.
template <typename E, int D>
__global__ void __launch_bounds__(256) paged_merge_kernel(const PgAttnArgs a, const PgParts p) {
  using Ty = PgType<E>;
  constexpr int DPL = D / 32;
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  const int t = (int)(row / a.Hq), h = (int)(row % a.Hq);
  if (a.cu && (t < a.cu[0] || t >= a.cu[a.R])) return;  // a padded row stays as it is
  float mx = -INFINITY;
  for (int z = lane; z < p.count; z += 32) mx = fmaxf(mx, p.lse[z * p.rows + row]);
  mx = warp_max(mx);
  float den = 0.f, o[DPL];
#pragma unroll
  for (int e = 0; e < DPL; ++e) o[e] = 0.f;
  for (int z0 = 0; z0 < p.count; z0 += 32) {
    const float ls = z0 + lane < p.count ? p.lse[(z0 + lane) * p.rows + row] : -INFINITY;
    const float wl = ls == -INFINITY ? 0.f : exp2f(ls - mx);
    for (int z = 0; z < min(32, p.count - z0); ++z) {
      const float w = __shfl_sync(0xffffffffu, wl, z);
      if (w == 0.f) continue;
      const float* src = p.o + ((z0 + z) * p.rows + row) * D + lane * DPL;
      float v[DPL];
      if constexpr (DPL == 2)
        *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(src);
      else
        *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
      den += w;
#pragma unroll
      for (int e = 0; e < DPL; ++e) o[e] = fmaf(w, v[e], o[e]);
    }
  }
  const float inv = den == 0.f ? 0.f : 1.f / den;  // NaN stays NaN
  E* dst = reinterpret_cast<E*>(a.out) + t * a.o_ts + (int64_t)h * a.o_hs + lane * DPL;
#pragma unroll
  for (int e = 0; e < DPL; e += 2)
    *reinterpret_cast<uint32_t*>(dst + e) = Ty::pack(o[e] * inv, o[e + 1] * inv);
}

int launch_paged_merge(const PgAttnArgs& a, bool bf16, const PgParts& parts, cudaStream_t s) {
  const int64_t blocks = (parts.rows + 7) / 8;
  if (blocks > 0x7fffffff) return DDQ_ERR_SHAPE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  cudaError_t e;
  if (bf16)
    e = a.c.D == 64 ? cudaLaunchKernelEx(&cfg, paged_merge_kernel<__nv_bfloat16, 64>, a, parts)
                    : cudaLaunchKernelEx(&cfg, paged_merge_kernel<__nv_bfloat16, 128>, a, parts);
  else
    e = a.c.D == 64 ? cudaLaunchKernelEx(&cfg, paged_merge_kernel<__half, 64>, a, parts)
                    : cudaLaunchKernelEx(&cfg, paged_merge_kernel<__half, 128>, a, parts);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return DDQ_ERR_LAUNCH;
  }
  return check_launch();
}

int launch_paged_attention(const PgAttnArgs& a, bool bf16, cudaStream_t s) {
  const int64_t blocks = ((int64_t)a.T * a.Hq + 7) / 8;
  if (blocks > 0x7fffffff) return DDQ_ERR_SHAPE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  cudaError_t e;
  if (bf16)
    e = a.c.D == 64 ? cudaLaunchKernelEx(&cfg, paged_attention_row_kernel<__nv_bfloat16, 64>, a)
                    : cudaLaunchKernelEx(&cfg, paged_attention_row_kernel<__nv_bfloat16, 128>, a);
  else
    e = a.c.D == 64 ? cudaLaunchKernelEx(&cfg, paged_attention_row_kernel<__half, 64>, a)
                    : cudaLaunchKernelEx(&cfg, paged_attention_row_kernel<__half, 128>, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return DDQ_ERR_LAUNCH;
  }
  return check_launch();
}

}  // namespace ddq
