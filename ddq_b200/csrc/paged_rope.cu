// paged_rope.cu - rotary embedding of q and k and the write of k and v into
// the pages of a paged KV cache, for any mix of prompts and single tokens.
//
// For token row t of the q/k/v projection, at position p = positions[t], with
// slot = slots[t] (page slot / page_size, row slot % page_size; < 0: none):
//   q_out[t, h]           = rope(q_h, p)
//   k[page, g, row]       = rope(k_g, p)       v[page, g, row] = v_g
// rope(x)[d] = x[d] cos[p, d] + rotate_half(x)[d] sin[p, d], products and sum
// rounded in fp32, then once to the element type, as the dense cache's write
// rounds them (rope.cu).
//
// One thread per 16-byte piece: 8 dimensions of the first half of a head with
// the matching 8 of the second half, or 8 dimensions of a value row.  HBM
// bound: qkv read once, q, k and v written once, and the cos and sin rows of
// the positions.
#include "launch.cuh"
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace ddq {

struct PrArgs {
  PgCache c;
  const void* qkv;
  int64_t qkv_stride;
  const float* cos;  // [max_pos, D]
  const float* sin;
  int64_t max_pos;
  const int64_t* slots;
  const int64_t* positions;
  void* q_out;  // [T, Hq, D]
  int64_t T;
  int Hq;
};

template <typename E, int D>
__global__ void __launch_bounds__(256) paged_rope_kv_kernel(const PrArgs a) {
  using Ty = PgType<E>;
  constexpr int DH = D / 2;
  constexpr int PH = DH / 8;  // pieces per half head
  constexpr int VP = D / 8;   // pieces per value row
  ptx::pdl_wait();            // qkv comes from the projection just before
  ptx::pdl_launch_dependents();
  const int Hkv = a.c.Hkv;
  const int rot = (a.Hq + Hkv) * PH;
  const int per_tok = rot + Hkv * VP;
  const int64_t total = a.T * per_tok;
  const int64_t nslots = (int64_t)a.c.num_pages << a.c.page_shift;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = i / per_tok;
    const int j = (int)(i - t * per_tok);
    const E* row = reinterpret_cast<const E*>(a.qkv) + t * a.qkv_stride;
    const bool is_q = j < a.Hq * PH;
    int64_t off = 0;  // of the cache row
    if (!is_q) {
      const int64_t slot = a.slots[t];
      if (slot < 0) continue;
      if (slot >= nslots) {
        record_device_error(DDQ_ERR_PAGE);
        continue;
      }
      off = (slot >> a.c.page_shift) * a.c.page_stride +
            (slot & ((1 << a.c.page_shift) - 1)) * a.c.row_stride;
    }
    if (j < rot) {
      const int h = j / PH, d0 = 8 * (j % PH);  // q heads, then k heads
      const int64_t p = a.positions[t];
      if (p < 0 || p >= a.max_pos) {
        record_device_error(DDQ_ERR_PAGE);
        continue;
      }
      const uint4 u1 = *reinterpret_cast<const uint4*>(row + (size_t)h * D + d0);
      const uint4 u2 = *reinterpret_cast<const uint4*>(row + (size_t)h * D + DH + d0);
      const float* cr = a.cos + p * D;
      const float* sr = a.sin + p * D;
      float c1[8], s1[8], c2[8], s2[8];
      *reinterpret_cast<float4*>(c1) = *reinterpret_cast<const float4*>(cr + d0);
      *reinterpret_cast<float4*>(c1 + 4) = *reinterpret_cast<const float4*>(cr + d0 + 4);
      *reinterpret_cast<float4*>(s1) = *reinterpret_cast<const float4*>(sr + d0);
      *reinterpret_cast<float4*>(s1 + 4) = *reinterpret_cast<const float4*>(sr + d0 + 4);
      *reinterpret_cast<float4*>(c2) = *reinterpret_cast<const float4*>(cr + DH + d0);
      *reinterpret_cast<float4*>(c2 + 4) = *reinterpret_cast<const float4*>(cr + DH + d0 + 4);
      *reinterpret_cast<float4*>(s2) = *reinterpret_cast<const float4*>(sr + DH + d0);
      *reinterpret_cast<float4*>(s2 + 4) = *reinterpret_cast<const float4*>(sr + DH + d0 + 4);
      const uint32_t w1[4] = {u1.x, u1.y, u1.z, u1.w}, w2[4] = {u2.x, u2.y, u2.z, u2.w};
      uint32_t o1[4], o2[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 x1 = Ty::to_f2(w1[e]), x2 = Ty::to_f2(w2[e]);
        o1[e] = Ty::pack(
            __fadd_rn(__fmul_rn(x1.x, c1[2 * e]), __fmul_rn(-x2.x, s1[2 * e])),
            __fadd_rn(__fmul_rn(x1.y, c1[2 * e + 1]), __fmul_rn(-x2.y, s1[2 * e + 1])));
        o2[e] = Ty::pack(
            __fadd_rn(__fmul_rn(x2.x, c2[2 * e]), __fmul_rn(x1.x, s2[2 * e])),
            __fadd_rn(__fmul_rn(x2.y, c2[2 * e + 1]), __fmul_rn(x1.y, s2[2 * e + 1])));
      }
      E* dst = is_q ? reinterpret_cast<E*>(a.q_out) + ((size_t)t * a.Hq + h) * D
                    : reinterpret_cast<E*>(a.c.k) + off + (int64_t)(h - a.Hq) * a.c.head_stride;
      *reinterpret_cast<uint4*>(dst + d0) = make_uint4(o1[0], o1[1], o1[2], o1[3]);
      *reinterpret_cast<uint4*>(dst + DH + d0) = make_uint4(o2[0], o2[1], o2[2], o2[3]);
    } else {
      const int jv = j - rot, g = jv / VP, d0 = 8 * (jv % VP);
      const uint4 u = *reinterpret_cast<const uint4*>(row + (size_t)(a.Hq + Hkv + g) * D + d0);
      *reinterpret_cast<uint4*>(reinterpret_cast<E*>(a.c.v) + off +
                                (int64_t)g * a.c.head_stride + d0) = u;
    }
  }
}

int launch_paged_rope_kv(const void* qkv, int64_t qkv_stride, const PgCache& c, bool bf16,
                         const float* cos, const float* sin, int64_t max_pos,
                         const int64_t* slots, const int64_t* positions, void* q_out, int64_t T,
                         int Hq, cudaStream_t s) {
  PrArgs a{c, qkv, qkv_stride, cos, sin, max_pos, slots, positions, q_out, T, Hq};
  const int per_tok = (Hq + c.Hkv) * (c.D / 16) + c.Hkv * (c.D / 8);
  const int sms = device_sm_count(current_device());
  if (sms <= 0) return DDQ_ERR_DEVICE;
  int64_t blocks = (T * per_tok + 255) / 256;
  if (blocks > (int64_t)sms * 8) blocks = (int64_t)sms * 8;
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
    e = c.D == 64 ? cudaLaunchKernelEx(&cfg, paged_rope_kv_kernel<__nv_bfloat16, 64>, a)
                  : cudaLaunchKernelEx(&cfg, paged_rope_kv_kernel<__nv_bfloat16, 128>, a);
  else
    e = c.D == 64 ? cudaLaunchKernelEx(&cfg, paged_rope_kv_kernel<__half, 64>, a)
                  : cudaLaunchKernelEx(&cfg, paged_rope_kv_kernel<__half, 128>, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return DDQ_ERR_LAUNCH;
  }
  return check_launch();
}

}  // namespace ddq
