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
// HBM bound: qkv read once, q, k and v written once, and the cos and sin rows of
// the positions.  A CTA takes a token at a time (several where a token has few
// pieces); a thread takes 8 dimensions of the first half of one or more heads
// with the matching 8 of the second half - always the same dimensions, so that
// the token's cos and sin stay in its registers for all its heads (32 bytes each
// were read again for every head: 204 us instead of 137, 6.1 TB/s, for 32768 tokens
// of 32 + 2 x 8 heads of 128) - and its 16-byte loads of all heads are in flight together.
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

constexpr int PR_NT = 128;
constexpr int PR_CTAS = 4;            // per SM: as many as are resident (16: 137 us, any number: 154)

template <typename E, int D>
__global__ void __launch_bounds__(PR_NT) paged_rope_kv_kernel(const PrArgs a) {
  using Ty = PgType<E>;
  constexpr int DH = D / 2;
  constexpr int PH = DH / 8;          // pieces per half head
  constexpr int HS = PR_NT / PH;      // heads a pass (PH threads each)
  constexpr int MAXP = 4;             // heads in flight per thread
  ptx::pdl_wait();                    // qkv comes from the projection just before
  ptx::pdl_launch_dependents();
  const int Hkv = a.c.Hkv, rot = a.Hq + Hkv, heads = rot + Hkv;
  const int d0 = 8 * (threadIdx.x % PH), hs = threadIdx.x / PH;
  const int64_t nslots = (int64_t)a.c.num_pages << a.c.page_shift;
  // work item: a token and one of its groups of HS * MAXP heads
  const int groups = (heads + HS * MAXP - 1) / (HS * MAXP);
  const int64_t items = a.T * groups;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t t = groups == 1 ? it : it / groups;
    const int h0 = (groups == 1 ? 0 : (int)(it - t * groups) * HS * MAXP) + hs;
    const E* row = reinterpret_cast<const E*>(a.qkv) + t * a.qkv_stride + d0;
    uint4 u1[MAXP], u2[MAXP];
#pragma unroll
    for (int i = 0; i < MAXP; ++i) {
      const int h = h0 + i * HS;
      if (h < heads) {
        u1[i] = *reinterpret_cast<const uint4*>(row + (size_t)h * D);
        u2[i] = *reinterpret_cast<const uint4*>(row + (size_t)h * D + DH);
      }
    }
    const int64_t p = a.positions[t], slot = a.slots[t];
    const bool turn = p >= 0 && p < a.max_pos, keep = slot >= 0 && slot < nslots;
    if ((!turn || slot >= nslots) && threadIdx.x == 0) record_device_error(DDQ_ERR_PAGE);
    float c1[8], s1[8], c2[8], s2[8];
    if (turn) {
      const float* cr = a.cos + p * D + d0;
      const float* sr = a.sin + p * D + d0;
      *reinterpret_cast<float4*>(c1) = *reinterpret_cast<const float4*>(cr);
      *reinterpret_cast<float4*>(c1 + 4) = *reinterpret_cast<const float4*>(cr + 4);
      *reinterpret_cast<float4*>(s1) = *reinterpret_cast<const float4*>(sr);
      *reinterpret_cast<float4*>(s1 + 4) = *reinterpret_cast<const float4*>(sr + 4);
      *reinterpret_cast<float4*>(c2) = *reinterpret_cast<const float4*>(cr + DH);
      *reinterpret_cast<float4*>(c2 + 4) = *reinterpret_cast<const float4*>(cr + DH + 4);
      *reinterpret_cast<float4*>(s2) = *reinterpret_cast<const float4*>(sr + DH);
      *reinterpret_cast<float4*>(s2 + 4) = *reinterpret_cast<const float4*>(sr + DH + 4);
    }
    const int64_t off = keep ? (slot >> a.c.page_shift) * a.c.page_stride +
                                   (slot & ((1 << a.c.page_shift) - 1)) * a.c.row_stride + d0
                             : 0;
#pragma unroll
    for (int i = 0; i < MAXP; ++i) {
      const int h = h0 + i * HS;
      if (h >= heads) break;
      E* dst;
      if (h < a.Hq) {
        if (!turn) continue;
        dst = reinterpret_cast<E*>(a.q_out) + ((size_t)t * a.Hq + h) * D + d0;
      } else if (h < rot) {
        if (!turn || !keep) continue;
        dst = reinterpret_cast<E*>(a.c.k) + off + (int64_t)(h - a.Hq) * a.c.head_stride;
      } else {
        if (!keep) continue;
        dst = reinterpret_cast<E*>(a.c.v) + off + (int64_t)(h - rot) * a.c.head_stride;
      }
      uint4 o1 = u1[i], o2 = u2[i];
      if (h < rot) {
        const uint32_t w1[4] = {u1[i].x, u1[i].y, u1[i].z, u1[i].w};
        const uint32_t w2[4] = {u2[i].x, u2[i].y, u2[i].z, u2[i].w};
        uint32_t r1[4], r2[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x1 = Ty::to_f2(w1[e]), x2 = Ty::to_f2(w2[e]);
          r1[e] = Ty::pack(
              __fadd_rn(__fmul_rn(x1.x, c1[2 * e]), __fmul_rn(-x2.x, s1[2 * e])),
              __fadd_rn(__fmul_rn(x1.y, c1[2 * e + 1]), __fmul_rn(-x2.y, s1[2 * e + 1])));
          r2[e] = Ty::pack(
              __fadd_rn(__fmul_rn(x2.x, c2[2 * e]), __fmul_rn(x1.x, s2[2 * e])),
              __fadd_rn(__fmul_rn(x2.y, c2[2 * e + 1]), __fmul_rn(x1.y, s2[2 * e + 1])));
        }
        o1 = make_uint4(r1[0], r1[1], r1[2], r1[3]);
        o2 = make_uint4(r2[0], r2[1], r2[2], r2[3]);
      }
      *reinterpret_cast<uint4*>(dst) = o1;
      *reinterpret_cast<uint4*>(dst + DH) = o2;
    }
  }
}

int launch_paged_rope_kv(const void* qkv, int64_t qkv_stride, const PgCache& c, bool bf16,
                         const float* cos, const float* sin, int64_t max_pos,
                         const int64_t* slots, const int64_t* positions, void* q_out, int64_t T,
                         int Hq, cudaStream_t s) {
  PrArgs a{c, qkv, qkv_stride, cos, sin, max_pos, slots, positions, q_out, T, Hq};
  const int per = PR_NT / (c.D / 16) * 4;  // heads of a work item
  const int64_t items = T * ((Hq + 2 * c.Hkv + per - 1) / per);
  const int sms = device_sm_count(current_device());
  if (sms <= 0) return DDQ_ERR_DEVICE;
  int64_t blocks = items;
  if (blocks > (int64_t)sms * PR_CTAS) blocks = (int64_t)sms * PR_CTAS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(PR_NT);
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
