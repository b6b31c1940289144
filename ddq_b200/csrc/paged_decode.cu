// paged_decode.cu - paged attention of one token per sequence over the
// sequence's own pages, joined with the part of a shared prefix.  Scores, cap,
// bias and softmax as paged_tc.cu states them, all keys of the sequence attended.
//
// HBM bound: every key and value is read once for the heads that share it, and
// sequences differ in length by orders of magnitude.  So the work is a flat
// list of units of 128 keys - sequence, key/value head (and group of 16 query
// heads), unit of the sequence - which the CTAs, as many as fit the GPU, share
// out evenly: CTA i of N takes units [i U / N, (i + 1) U / N), whatever
// sequences they belong to.  The list is never stored: each CTA sums the
// lengths (4 bytes a sequence) and finds its first unit.  Where a CTA's range
// cuts a sequence, its part goes to one of two side slots of the CTA, and the
// joining kernel adds the parts up in order; there are no atomics.
//
// Four warps, 32 keys each per unit, each with a ring of its own that TMA fills
// from the pages DC_DEPTH units ahead, across the ends of sequences.  Per 32
// keys, on mma.sync m16n8k16 with the keys (and the head dimensions) on the 16
// rows, the 8 columns being query heads:
//   S^T[key, head]  = K q^T            ldmatrix of K as it lies
//   O^T[dim, head] += V^T P^T          ldmatrix.trans of V as it lies; P^T from
//                                      the accumulator layout by movmatrix
// so that up to 8 heads waste nothing, and each lane keeps the maximum, the sum
// and the outputs of the same two heads.
#include <cudaTypedefs.h>

#include "launch.cuh"
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace ddq {

constexpr int DC_NW = 4;
constexpr int DC_UNIT = 32 * DC_NW;  // keys
constexpr int DC_DEPTH = 3;
constexpr int DC_SCAN = 64;          // sequences a thread sums at most
constexpr int DC_MAXB = DC_SCAN * DC_NW * 32;

// Side slots (2 per CTA), and for each segment (sequence, key/value head, head
// group) the CTAs that hold its first and its last unit.
struct DcSide {
  float* o;      // [2 N][heads][D]
  float* lse;    // [2 N][heads]
  int2* seg;     // [B * Hkv * groups]
};

template <int D, int NB>
struct DcSmem {
  uint8_t ring[DC_NW * DC_DEPTH][2][32 * D * 2];
  float acc[DC_NW][8 * NB][D];
  float m[DC_NW][8 * NB], l[DC_NW][8 * NB];
  unsigned long long full[DC_NW * DC_DEPTH];
  long long wsum[DC_NW];
  int start[4];
  int abort_flag;
};

__device__ __forceinline__ float dc_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void dc_ldsm(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void dc_ldsm_t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ uint32_t dc_transpose(uint32_t x) {  // 8 x 8 16-bit elements
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <typename E>
__device__ __forceinline__ void dc_mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void dc_mma<__half>(float* d, const uint32_t* a, uint32_t b0,
                                               uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void dc_mma<__nv_bfloat16>(float* d, const uint32_t* a, uint32_t b0,
                                                      uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// byte offset of 16-byte piece j of row r in a tile of 64 elements a row
__device__ __forceinline__ uint32_t dc_swz(int r, int j) { return r * 128 + ((j ^ (r & 7)) << 4); }

__host__ __device__ __forceinline__ int dc_groups(int G) { return (G + 15) / 16; }

// A position in the list of units.
struct DcWalk {
  int b, seg, c;   // sequence, key/value head and head group, unit of the sequence
  int len, units;  // of the sequence
};

template <typename E, int D, int NB>
__global__ void __launch_bounds__(DC_NW * 32)
    paged_decode_kernel(const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v, const PgAttnArgs a,
                        const PgParts parts, const DcSide side, const unsigned long long tmo) {
  using Ty = PgType<E>;
  using Sm = DcSmem<D, NB>;
  constexpr int H2 = D / 64;
  constexpr float LOG2E = 1.4426950408889634f;
  extern __shared__ uint8_t dc_raw[];
  Sm& sm = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(dc_raw) + 1023) &
                                  ~static_cast<uintptr_t>(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row4 = lane >> 2, col2 = 2 * (lane & 3);
  const int G = a.Hq / a.c.Hkv, groups = dc_groups(G), segs = a.c.Hkv * groups;
  const bool prefix = a.prefix_len > 0;
  if (tid == 0) {
    for (int s = 0; s < DC_NW * DC_DEPTH; ++s) ptx::mbar_init(ptx::smem_u32(&sm.full[s]), 1);
    sm.abort_flag = 0;
    sm.start[0] = -1;
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tm_k);
    ptx::prefetch_tmap(&tm_v);
  }
  // Behind the prefix kernel nothing that it writes is read here, and it let
  // this kernel start only after its own wait: q, the pages and the lengths are
  // there.  The wait comes before the exit, so that this kernel's end implies
  // the prefix kernel's.
  if (!prefix) ptx::pdl_wait();
  ptx::pdl_launch_dependents();

  // ---- this CTA's units
  auto units_of = [&](int len) { return max(1, (len + DC_UNIT - 1) / DC_UNIT); };
  const int per = (a.R + DC_NW * 32 - 1) / (DC_NW * 32);  // sequences a thread sums
  const int b0 = min(tid * per, a.R), b1 = min(b0 + per, a.R);
  long long sum = 0;
  for (int b = b0; b < b1; ++b) sum += units_of(pg_len(a, b));
  long long inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) sm.wsum[warp] = inc;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < DC_NW; ++w) {
    if (w < warp) inc += sm.wsum[w];
    total += sm.wsum[w];
  }
  total *= segs;
  // (with fewer units than CTAs the first `total` take one each: the parts of a
  // sequence lie in consecutive CTAs, none of them empty)
  const long long N = min((long long)gridDim.x, total);
  const long long u0 = total * blockIdx.x / N, u1 = total * (blockIdx.x + 1) / N;
  if (blockIdx.x >= N) {
    if (prefix) ptx::pdl_wait();
    return;
  }
  long long at = (inc - sum) * segs;
  if (u0 >= at && u0 < inc * segs) {
    int b = b0, n = units_of(pg_len(a, b));
    while (u0 >= at + (long long)n * segs) {
      at += (long long)n * segs;
      n = units_of(pg_len(a, ++b));
    }
    sm.start[0] = b;
    sm.start[1] = (int)((u0 - at) / n);
    sm.start[2] = (int)((u0 - at) % n);
  }
  __syncthreads();
  auto load_len = [&](DcWalk& w) {
    w.len = w.b < a.R ? pg_len(a, w.b) : 0;
    w.units = units_of(w.len);
  };
  auto advance = [&](DcWalk& w) {
    if (++w.c < w.units) return;
    w.c = 0;
    if (++w.seg < segs) return;
    w.seg = 0;
    ++w.b;
    load_len(w);
  };
  DcWalk cw{sm.start[0], sm.start[1], sm.start[2], 0, 0};
  load_len(cw);
  const int count = (int)(u1 - u0);

  // ---- loads: chunk after chunk of this warp, the page numbers one ahead
  const int br = min(1 << a.c.page_shift, 32), nb = 32 / br;  // rows of a box, boxes of 32 keys
  const int sub = lane % nb, dh = (lane / nb) % H2, kv = lane / (nb * H2);
  const uint32_t ring = ptx::smem_u32(&sm.ring[warp * DC_DEPTH][0][0]);
  const uint32_t bar = ptx::smem_u32(&sm.full[warp * DC_DEPTH]);
  DcWalk lw = cw;
  int ahead = 0;        // units that lw is past u0
  int issued = 0;       // chunks requested
  int pend_page = 0, pend_row = 0, pend_head = 0;
  bool pend_mine = false, pend = false;
  auto look = [&] {     // the next chunk with keys: its page number, not used yet
    pend = false;
    while (ahead < count) {
      const int base = lw.c * DC_UNIT + warp * 32;
      if (base < lw.len) {
        const int key = base + sub * br;
        pend_mine = kv < 2 && key < lw.len;
        if (pend_mine)
          pend_page = a.table[lw.b * a.table_stride + (key >> a.c.page_shift)];
        pend_row = key & ((1 << a.c.page_shift) - 1);
        pend_head = lw.seg / groups;
        pend = true;
        advance(lw);
        ++ahead;
        return;
      }
      advance(lw);
      ++ahead;
    }
  };
  auto issue = [&] {    // the chunk looked up into the next slot
    const int s = issued % DC_DEPTH;
    bool mine = pend_mine;
    if (mine) mine = pg_check(a.c, pend_page) >= 0;
    const uint32_t bytes = (uint32_t)__popc(__ballot_sync(0xffffffffu, mine)) * br * 128u;
    if (lane == 0) ptx::mbar_arrive_expect_tx(bar + 8 * s, bytes);
    __syncwarp();
    if (mine)
      ptx::tma_load_4d(ring + (uint32_t)(((s * 2 + kv) * H2 + dh) * 4096 + sub * br * 128),
                       kv ? &tm_v : &tm_k, dh * 64, pend_row, pend_head, pend_page, bar + 8 * s);
    ++issued;
  };
  look();
  for (int i = 0; i < DC_DEPTH && pend; ++i) {
    issue();
    look();
  }

  // ---- compute
  const bool plain = a.cap == 0.f && a.slopes == nullptr && a.scale > 0.f;
  const float mul = plain ? a.scale * LOG2E : 1.f;
  uint32_t q[NB][D / 16][2];
  float m[NB][2], l[NB][2], slope[NB][2], o[D / 16][NB][4];
  // the queries of a segment, requested while the segment before it is joined
  auto load_q = [&](const DcWalk& w) {
    const int grp = w.seg % groups, heads = min(16, G - grp * 16);
    const E* base = reinterpret_cast<const E*>(a.q) + w.b * a.q_ts + col2;
    const int first = w.seg / groups * G + grp * 16;
#pragma unroll
    for (int nbk = 0; nbk < NB; ++nbk) {
      const int hq = row4 + 8 * nbk;
      const E* src = base + (int64_t)(first + hq) * a.q_hs;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) {
        q[nbk][e][0] = hq < heads ? *reinterpret_cast<const uint32_t*>(src + 16 * e) : 0u;
        q[nbk][e][1] = hq < heads ? *reinterpret_cast<const uint32_t*>(src + 16 * e + 8) : 0u;
      }
    }
  };
  load_q(cw);
  bool fresh = true;      // the next unit starts a part of a segment
  bool whole = true;      // ... which begins in this CTA
  int used = 0;
  bool dead = false;
  for (int u = 0; u < count; ++u) {
    const int g = cw.seg / groups, h0 = g * G + (cw.seg % groups) * 16;  // first query head
    const int heads = min(16, G - (cw.seg % groups) * 16);
    if (fresh) {
      fresh = false;
      whole = cw.c == 0;
#pragma unroll
      for (int nbk = 0; nbk < NB; ++nbk) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          m[nbk][x] = -INFINITY;
          l[nbk][x] = 0.f;
          const int hs = col2 + x + 8 * nbk;
          slope[nbk][x] = a.slopes && hs < heads ? a.slopes[h0 + hs] * LOG2E : 0.f;
        }
#pragma unroll
        for (int e = 0; e < D / 16; ++e)
          o[e][nbk][0] = o[e][nbk][1] = o[e][nbk][2] = o[e][nbk][3] = 0.f;
      }
    }
    const int base = cw.c * DC_UNIT + warp * 32;
    const int have = min(32, cw.len - base);
    if (have > 0 && !dead) {
      const int s = used % DC_DEPTH;
      dead = !__all_sync(0xffffffffu, ptx::mbar_wait(bar + 8 * s, (uint32_t)(used / DC_DEPTH) & 1u,
                                                     tmo, &sm.abort_flag));
      if (!dead) {
        const uint32_t ks = ring + (uint32_t)(s * 2 * H2 * 4096), vs = ks + H2 * 4096;
        if (have < 32) {  // rows behind the last key may hold anything: 0 x NaN is NaN
          uint8_t* vr = &sm.ring[warp * DC_DEPTH + s][1][0];
          for (int x = have * 8 + lane; x < 32 * 8; x += 32)
#pragma unroll
            for (int hb = 0; hb < H2; ++hb)
              *reinterpret_cast<uint4*>(vr + hb * 4096 + x * 16) = make_uint4(0u, 0u, 0u, 0u);
          __syncwarp();
        }
        // S^T: keys 16 mt + row4 (+ 8), heads col2 (+ 1)
        float sc[2][NB][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
          for (int nbk = 0; nbk < NB; ++nbk)
            sc[mt][nbk][0] = sc[mt][nbk][1] = sc[mt][nbk][2] = sc[mt][nbk][3] = 0.f;
#pragma unroll
          for (int e = 0; e < D / 16; ++e) {
            uint32_t r[4];
            dc_ldsm(ks + (e >> 2) * 4096 +
                        dc_swz(16 * mt + (lane & 15), 2 * (e & 3) + (lane >> 4)), r);
#pragma unroll
            for (int nbk = 0; nbk < NB; ++nbk)
              dc_mma<E>(sc[mt][nbk], r, q[nbk][e][0], q[nbk][e][1]);
          }
        }
        bool grow = false;
        float mx[NB][2];
#pragma unroll
        for (int nbk = 0; nbk < NB; ++nbk)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            mx[nbk][x] = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                float& v = sc[mt][nbk][2 * y + x];
                const int key = 16 * mt + row4 + 8 * y;
                if (!plain) {
                  if (a.cap > 0.f) {  // cap - 2 cap / (exp(2 y / cap) + 1), as paged_tc.cu
                    const float A = a.cap * LOG2E;
                    v = A - __fdividef(2.f * A, dc_exp2(v * (2.f * LOG2E * a.scale / a.cap)) + 1.f);
                  } else {
                    v *= a.scale * LOG2E;
                  }
                  v = fmaf(-slope[nbk][x], (float)(cw.len - 1 - base - key), v);
                }
                v = key < have ? v * mul : -INFINITY;
                mx[nbk][x] = fmaxf(mx[nbk][x], v);
              }
            grow |= mx[nbk][x] > m[nbk][x] + 8.f;
          }
        if (__any_sync(0xffffffffu, grow)) {  // move the maxima, rescale
#pragma unroll
          for (int nbk = 0; nbk < NB; ++nbk) {
            float al[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float v = mx[nbk][x];
#pragma unroll
              for (int sh = 4; sh < 32; sh <<= 1)
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, sh));
              const float mn = fmaxf(m[nbk][x], v);
              al[x] = m[nbk][x] == -INFINITY ? 1.f : dc_exp2(m[nbk][x] - mn);  // o is 0 before
              m[nbk][x] = mn;
              l[nbk][x] *= al[x];
            }
#pragma unroll
            for (int e = 0; e < D / 16; ++e) {
              o[e][nbk][0] *= al[0];
              o[e][nbk][1] *= al[1];
              o[e][nbk][2] *= al[0];
              o[e][nbk][3] *= al[1];
            }
          }
        }
        uint32_t pb[2][NB][2];  // P^T of 16 keys: B fragments
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int nbk = 0; nbk < NB; ++nbk) {
            const float m0 = m[nbk][0] == -INFINITY ? 0.f : m[nbk][0];
            const float m1 = m[nbk][1] == -INFINITY ? 0.f : m[nbk][1];
            const float p0 = dc_exp2(sc[mt][nbk][0] - m0), p1 = dc_exp2(sc[mt][nbk][1] - m1);
            const float p2 = dc_exp2(sc[mt][nbk][2] - m0), p3 = dc_exp2(sc[mt][nbk][3] - m1);
            l[nbk][0] += p0 + p2;
            l[nbk][1] += p1 + p3;
            pb[mt][nbk][0] = dc_transpose(Ty::pack(p0, p1));
            pb[mt][nbk][1] = dc_transpose(Ty::pack(p2, p3));
          }
        // O^T: dims 16 e + row4 (+ 8), heads col2 (+ 1)
#pragma unroll
        for (int e = 0; e < D / 16; ++e)
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            uint32_t r[4];
            dc_ldsm_t(vs + (e >> 2) * 4096 + dc_swz(16 * mt + (lane & 7) + 8 * (lane >> 4),
                                                    2 * (e & 3) + ((lane >> 3) & 1)), r);
#pragma unroll
            for (int nbk = 0; nbk < NB; ++nbk)
              dc_mma<E>(o[e][nbk], r, pb[mt][nbk][0], pb[mt][nbk][1]);
          }
        ++used;
        // the slot is free: the next chunk into it
        __syncwarp();
        if (pend) {
          ptx::fence_proxy_async_smem();
          issue();
          look();
        }
      }
    }

    const DcWalk now = cw;
    advance(cw);
    if (cw.c != 0 && u + 1 < count) continue;
    // ---- the end of this CTA's part of the segment: the warps' results, joined
    fresh = true;
    if (u + 1 < count) load_q(cw);
#pragma unroll
    for (int nbk = 0; nbk < NB; ++nbk)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float v = l[nbk][x];
#pragma unroll
        for (int sh = 4; sh < 32; sh <<= 1) v += __shfl_xor_sync(0xffffffffu, v, sh);
        if (row4 == 0) {
          sm.m[warp][8 * nbk + col2 + x] = m[nbk][x];
          sm.l[warp][8 * nbk + col2 + x] = v;
        }
#pragma unroll
        for (int e = 0; e < D / 16; ++e) {
          sm.acc[warp][8 * nbk + col2 + x][16 * e + row4] = o[e][nbk][x];
          sm.acc[warp][8 * nbk + col2 + x][16 * e + row4 + 8] = o[e][nbk][2 + x];
        }
      }
    __syncthreads();
    const bool done = now.c == now.units - 1;     // the part has the segment's last unit
    const bool full = whole && done;
    if (tid == 0) {
      int2* info = side.seg + (int64_t)now.b * segs + now.seg;
      if (whole) info->x = blockIdx.x;
      if (done) info->y = blockIdx.x;
    }
    const int slot = 2 * blockIdx.x + (whole ? 1 : 0);
    for (int i = tid; i < heads * (D / 2); i += DC_NW * 32) {
      const int h = i / (D / 2), d = 2 * (i % (D / 2));
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < DC_NW; ++w) top = fmaxf(top, sm.m[w][h]);
      float den = 0.f, v0 = 0.f, v1 = 0.f;
#pragma unroll
      for (int w = 0; w < DC_NW; ++w) {
        const float lw_ = sm.l[w][h];
        if (lw_ == 0.f) continue;  // no keys (a NaN goes on)
        const float c = dc_exp2(sm.m[w][h] == top ? 0.f : sm.m[w][h] - top);
        const float2 av = *reinterpret_cast<const float2*>(&sm.acc[w][h][d]);
        den = fmaf(lw_, c, den);
        v0 = fmaf(av.x, c, v0);
        v1 = fmaf(av.y, c, v1);
      }
      const float inv = den == 0.f ? 0.f : 1.f / den;
      const float lse = den == 0.f ? -INFINITY : top + log2f(den);
      const int64_t row = (int64_t)now.b * a.Hq + h0 + h;
      if (full && !prefix) {
        *reinterpret_cast<uint32_t*>(reinterpret_cast<E*>(a.out) + now.b * a.o_ts +
                                     (int64_t)(h0 + h) * a.o_hs + d) = Ty::pack(v0 * inv, v1 * inv);
      } else if (full) {
        const int64_t pr = (int64_t)(parts.count - 1) * parts.rows + row;
        *reinterpret_cast<float2*>(parts.o + pr * D + d) = make_float2(v0 * inv, v1 * inv);
        if (d == 0) parts.lse[pr] = lse;
      } else {
        const int64_t pr = (int64_t)slot * 16 + h;
        *reinterpret_cast<float2*>(side.o + pr * D + d) = make_float2(v0 * inv, v1 * inv);
        if (d == 0) side.lse[pr] = lse;
      }
    }
    __syncthreads();  // acc, m and l are free again
  }
  if (dead) {         // copies in flight land before the shared memory goes
    for (int k = used; k < issued; ++k) {
      const long long t0 = clock64();
      while (!ptx::mbar_try_wait(bar + 8 * (k % DC_DEPTH), (uint32_t)(k / DC_DEPTH) & 1u))
        if (clock64() - t0 > (long long)(tmo * 2ull)) break;
    }
    if (lane == 0) pg_error(a.c, DDQ_ERR_TIMEOUT);
  }
  if (prefix) ptx::pdl_wait();
}

// Joins the parts of every row, in order: the prefix splits, then the own keys
// (whole, or the side slots of the CTAs that share them).
//   o = sum_z 2^(lse_z - max) o_z / sum_z 2^(lse_z - max)
// One warp per row.
template <typename E, int D>
__global__ void __launch_bounds__(256)
    paged_decode_merge_kernel(const PgAttnArgs a, const PgParts p, const DcSide side) {
  using Ty = PgType<E>;
  constexpr int DPL = D / 32;
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= (int64_t)a.T * a.Hq) return;
  const int b = (int)(row / a.Hq), h = (int)(row % a.Hq);
  const int G = a.Hq / a.c.Hkv, groups = dc_groups(G);
  const int g = h / G, hh = h % G;
  const int2 ends = side.seg[((int64_t)b * a.c.Hkv + g) * groups + hh / 16];
  const bool split = ends.x != ends.y;
  if (!split && p.count == 0) return;  // written already
  // parts 0 .. p.count - 2: prefix; p.count - 1: own keys, unless split
  const int first = split ? max(p.count - 1, 0) : p.count;
  const int n = first + (split ? ends.y - ends.x + 1 : 0);
  auto index = [&](int z) {  // side slot of part z
    const int cta = ends.x + (z - first);
    return (int64_t)(2 * cta + (z == first ? 1 : 0)) * 16 + hh % 16;
  };
  auto lse_of = [&](int z) {
    return z >= n ? -INFINITY : z < first ? p.lse[z * p.rows + row] : side.lse[index(z)];
  };
  float mx = -INFINITY;
  for (int z = lane; z < n; z += 32) mx = fmaxf(mx, lse_of(z));
  mx = warp_max(mx);
  float den = 0.f, o[DPL];
#pragma unroll
  for (int e = 0; e < DPL; ++e) o[e] = 0.f;
  for (int z0 = 0; z0 < n; z0 += 32) {
    const float ls = lse_of(z0 + lane);
    const float wl = ls == -INFINITY ? 0.f : exp2f(ls - mx);
    const int m = min(32, n - z0);
    for (int z1 = 0; z1 < m; z1 += 4) {  // four parts in flight
      float v[4][DPL], w[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int z = z0 + z1 + y;
        w[y] = __shfl_sync(0xffffffffu, wl, (z1 + y) & 31);
        if (z >= n) w[y] = 0.f;
#pragma unroll
        for (int e = 0; e < DPL; ++e) v[y][e] = 0.f;
        if (w[y] != 0.f) {  // a part without keys was not written
          const float* src =
              (z < first ? p.o + (z * p.rows + row) * D : side.o + index(z) * D) + lane * DPL;
          if constexpr (DPL == 2)
            *reinterpret_cast<float2*>(v[y]) = *reinterpret_cast<const float2*>(src);
          else
            *reinterpret_cast<float4*>(v[y]) = *reinterpret_cast<const float4*>(src);
        }
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        den += w[y];
#pragma unroll
        for (int e = 0; e < DPL; ++e) o[e] = fmaf(w[y], v[y][e], o[e]);
      }
    }
  }
  const float inv = den == 0.f ? 0.f : 1.f / den;  // NaN stays NaN
  E* dst = reinterpret_cast<E*>(a.out) + b * a.o_ts + (int64_t)h * a.o_hs + lane * DPL;
#pragma unroll
  for (int e = 0; e < DPL; e += 2)
    *reinterpret_cast<uint32_t*>(dst + e) = Ty::pack(o[e] * inv, o[e + 1] * inv);
}

template <int D, int NB>
constexpr int dc_smem_bytes() { return (int)sizeof(DcSmem<D, NB>) + 1024; }

// CTAs that fit the GPU at once: two per SM with 64-wide heads (105 KB each).
int dc_ctas(int64_t B, int Hq, int Hkv, int D, int64_t keys, int sms) {
  const int64_t most = B * Hkv * dc_groups(Hq / Hkv) * ((keys + DC_UNIT - 1) / DC_UNIT);
  const int64_t fit = (int64_t)sms * (D == 64 ? 2 : 1);
  return (int)(most < 1 ? 1 : most < fit ? most : fit);
}

DcPlan dc_plan(int64_t B, int Hq, int Hkv, int D, int64_t keys, int64_t prefix, int sms) {
  DcPlan p;
  p.ctas = dc_ctas(B, Hq, Hkv, D, keys, sms);
  p.splits = prefix ? tc_splits(B, 1, Hq, Hkv, prefix, false, sms) : 0;
  const int64_t rows = B * Hq, count = prefix ? p.splits + 1 : 0;
  p.off_lse = (size_t)count * rows * D * 4;
  p.off_so = p.off_lse + ((size_t)count * rows * 4 + 15) / 16 * 16;
  p.off_sl = p.off_so + (size_t)p.ctas * 2 * 16 * D * 4;
  p.off_seg = p.off_sl + (size_t)p.ctas * 2 * 16 * 4;
  p.bytes = p.off_seg + (size_t)B * Hkv * dc_groups(Hq / Hkv) * sizeof(int2);
  return p;
}

int launch_paged_decode(const PgAttnArgs& a, bool bf16, void* ws, const DcPlan& plan,
                        unsigned long long tmo, cudaStream_t s) {
  if (a.R > DC_MAXB) return DDQ_ERR_SHAPE;
  uint8_t* w = static_cast<uint8_t*>(ws);
  const int count = a.prefix_len ? plan.splits + 1 : 0;
  const PgParts parts{count ? reinterpret_cast<float*>(w) : nullptr,
                      count ? reinterpret_cast<float*>(w + plan.off_lse) : nullptr,
                      (int64_t)a.T * a.Hq, 0, count};
  const DcSide side{reinterpret_cast<float*>(w + plan.off_so),
                    reinterpret_cast<float*>(w + plan.off_sl),
                    reinterpret_cast<int2*>(w + plan.off_seg)};
  int st = DDQ_OK;
  if (count) {
    st = launch_paged_tc(a, bf16, parts, plan.splits, tmo, s);
    if (st) return st;
  }
  CUtensorMap tk, tv;
  const int br = (1 << a.c.page_shift) < 32 ? (1 << a.c.page_shift) : 32;
  st = pg_tensor_map(&tk, a.c, a.c.k, bf16, br);
  if (!st) st = pg_tensor_map(&tv, a.c, a.c.v, bf16, br);
  if (st) return st;
  const int dev = current_device();
  static SmemAttrOnce attr[2][2][2];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)plan.ctas);
  cfg.blockDim = dim3(DC_NW * 32);
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaSuccess;
  auto go = [&](auto kern, SmemAttrOnce& once, int smem) -> int {
    const int ast = ensure_smem_attr(once, dev, kern, smem);
    if (ast) return ast;
    cfg.dynamicSmemBytes = smem;
    e = cudaLaunchKernelEx(&cfg, kern, tk, tv, a, parts, side, tmo);
    return DDQ_OK;
  };
  const bool wide = a.Hq / a.c.Hkv > 8;
#define DDQ_DC(D_, NB_)                                                                        \
  (bf16 ? go(paged_decode_kernel<__nv_bfloat16, D_, NB_>, attr[1][D_ / 128][NB_ - 1],          \
             dc_smem_bytes<D_, NB_>())                                                         \
        : go(paged_decode_kernel<__half, D_, NB_>, attr[0][D_ / 128][NB_ - 1],                 \
             dc_smem_bytes<D_, NB_>()))
  if (a.c.D == 64)
    st = wide ? DDQ_DC(64, 2) : DDQ_DC(64, 1);
  else
    st = wide ? DDQ_DC(128, 2) : DDQ_DC(128, 1);
#undef DDQ_DC
  if (st) return st;
  if (e == cudaSuccess) {
    cfg.gridDim = dim3((unsigned)(((int64_t)a.T * a.Hq + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    if (bf16)
      e = a.c.D == 64
              ? cudaLaunchKernelEx(&cfg, paged_decode_merge_kernel<__nv_bfloat16, 64>, a, parts, side)
              : cudaLaunchKernelEx(&cfg, paged_decode_merge_kernel<__nv_bfloat16, 128>, a, parts, side);
    else
      e = a.c.D == 64
              ? cudaLaunchKernelEx(&cfg, paged_decode_merge_kernel<__half, 64>, a, parts, side)
              : cudaLaunchKernelEx(&cfg, paged_decode_merge_kernel<__half, 128>, a, parts, side);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return DDQ_ERR_LAUNCH;
  }
  return check_launch();
}

}  // namespace ddq
