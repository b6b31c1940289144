// paged_decode.cu - paged attention of one token per sequence over the
// sequence's own pages, joined with the part of a shared prefix.  Scores, cap,
// bias and softmax as paged_tc.cu states them, all keys of the sequence attended.
//
// HBM bound: every key and value is read once for the heads that share it, and
// sequences differ in length by orders of magnitude.  So the work is a flat
// list of units of 32 keys - sequence, key/value head (and group of 16 query
// heads), unit of the sequence - which the warps of as many CTAs as fit the GPU
// share out evenly: warp i of N takes units [i U / N, (i + 1) U / N), whatever
// sequences they belong to.  The list is never stored: each CTA sums the
// lengths (4 bytes a sequence) and finds its warps' first units.  Where a warp's
// range cuts a sequence, its part goes to one of two side slots of the warp, and
// the joining kernel adds the parts up in order; there are no atomics, and no
// warp waits for another one (with a CTA per range, its four warps joined at the
// end of every sequence, 2048 segments of 0 to 511 keys, 128-wide heads, took 77 us
// instead of 55; 40 sequences of 1 to 32768 keys take 284 us, 92% of a copy's rate).
//
// Each warp has a ring of its own, K and V of a unit in turn, that TMA fills from
// the pages, across the ends of sequences.  Per unit, on mma.sync m16n8k16 with the
// keys (and the head dimensions) on the 16 rows, the 8 columns being query heads:
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

constexpr int DC_NW = 8;             // warps: two a quarter of the SM hide each other's latency
constexpr int DC_UNIT = 32;          // keys
constexpr int DC_SLOTS = 3;          // of 32 rows of K or of V in turn, per warp
constexpr int DC_SCAN = 32;          // sequences a thread sums at most
constexpr int DC_MAXB = DC_SCAN * DC_NW * 32;

// Side slots (2 per warp), and for each segment (sequence, key/value head, head
// group) the warps that hold its first and its last unit.
struct DcSide {
  float* o;      // [2 N][16][D]
  float* lse;    // [2 N][16]
  int2* seg;     // [B * Hkv * groups]
};

template <int D>
struct DcSmem {
  uint8_t ring[DC_NW * DC_SLOTS][32 * D * 2];
  // a warp's results of 8 heads (4 where two CTAs shall fit) on their way out
  static constexpr int HEADS = D == 64 ? 4 : 8;
  float out[DC_NW][HEADS][D + 4];
  unsigned long long full[DC_NW * DC_SLOTS];
  long long wsum[DC_NW];
  int most[DC_NW];
  int start[DC_NW][6];
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

// CTAs of an SM, by registers and shared memory: 106 KB for 64-wide heads.  (With 8 heads
// on their way out at a time it was 115 KB, two CTAs did not fit, and the units, shared
// out for two an SM, ran as two waves: 64 sequences of 1 to 8192 keys, 14/2 heads of 64,
// in 40 us instead of 34.)
__host__ __device__ constexpr int dc_resident(int d, int nb) { return d == 64 && nb == 1 ? 2 : 1; }

__host__ __device__ __forceinline__ int dc_groups(int G) { return (G + 15) / 16; }

// A position in the list of units.
struct DcWalk {
  int b, g, grp, c;  // sequence, key/value head, head group, unit of the sequence
  int len, units;    // of the sequence
};

// x / d where x mostly fits 32 bits (a 64-bit division takes some 150 instructions)
__device__ __forceinline__ long long dc_div(long long x, long long d) {
  if (((x | d) >> 32) == 0) return (uint32_t)x / (uint32_t)d;
  return x / d;
}

template <typename E, int D, int NB>
__global__ void __launch_bounds__(DC_NW * 32, dc_resident(D, NB))
    paged_decode_kernel(const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v, const PgAttnArgs a,
                        const PgParts parts, const DcSide side, const unsigned long long tmo,
                        const int never) {
  using Ty = PgType<E>;
  using Sm = DcSmem<D>;
  constexpr int H2 = D / 64;
  constexpr float LOG2E = 1.4426950408889634f;
  extern __shared__ uint8_t dc_raw[];
  Sm& sm = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(dc_raw) + 1023) &
                                  ~static_cast<uintptr_t>(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row4 = lane >> 2, col2 = 2 * (lane & 3);
  const int G = a.G, groups = dc_groups(G), segs = a.c.Hkv * groups;
  const bool prefix = a.prefix_len > 0;
  if (tid == 0) {
    for (int s = 0; s < DC_NW * DC_SLOTS; ++s) ptx::mbar_init(ptx::smem_u32(&sm.full[s]), 1);
    sm.abort_flag = 0;
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

  // ---- this warp's units
  auto units_of = [&](int len) { return max(1, (len + DC_UNIT - 1) / DC_UNIT); };
  const int per = (a.R + DC_NW * 32 - 1) / (DC_NW * 32);  // sequences a thread sums
  const int b0 = min(tid * per, a.R), b1 = min(b0 + per, a.R);
  long long sum = 0;
  int most = 0;  // units of the longest sequence
  for (int b = b0; b < b1; ++b) {
    const int n = units_of(pg_len(a, b));
    sum += n;
    most = max(most, n);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  long long inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) {
    sm.wsum[warp] = inc;
    sm.most[warp] = most;
  }
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < DC_NW; ++w) {
    if (w < warp) inc += sm.wsum[w];
    total += sm.wsum[w];
    most = max(most, sm.most[w]);
  }
  total *= segs;
  // With few units the first warps take `least` each (the parts of a sequence lie
  // in consecutive warps, none of them empty): a unit more costs a warp 0.35 us, 32
  // parts more cost the joining 0.8 us, so least^2 = most / 14 or so.
  const int least = max(1, (int)(sqrtf((float)most * 0.0625f) + 0.5f));
  const long long N = max(1ll, min((long long)gridDim.x * DC_NW, total / least));
  const long long w0 = (long long)blockIdx.x * DC_NW;
  if (w0 >= N) {
    if (prefix) ptx::pdl_wait();
    return;
  }
  // warp i starts at unit i q + min(i, r): the first r take one more
  const long long uq = dc_div(total, N), ur = total - uq * N;
  for (int w = 0; w < DC_NW && w0 + w < N; ++w) {
    const long long u0 = (w0 + w) * uq + min(w0 + w, ur);
    long long at = (inc - sum) * segs;
    if (u0 < at || u0 >= inc * segs) continue;
    int b = b0, len = pg_len(a, b), n = units_of(len);
    while (u0 >= at + (long long)n * segs) {
      at += (long long)n * segs;
      len = pg_len(a, ++b);
      n = units_of(len);
    }
    const int seg = (int)dc_div(u0 - at, n);
    sm.start[w][0] = b;
    sm.start[w][1] = groups == 1 ? seg : seg / groups;
    sm.start[w][2] = groups == 1 ? 0 : seg % groups;
    sm.start[w][3] = (int)(u0 - at - (long long)seg * n);
    sm.start[w][4] = len;
    sm.start[w][5] = n;
  }
  __syncthreads();
  if (w0 + warp >= N) {
    if (prefix) ptx::pdl_wait();
    return;
  }
  const int worker = (int)w0 + warp;
  auto load_len = [&](DcWalk& w) {
    w.len = w.b < a.R ? pg_len(a, w.b) : 0;
    w.units = units_of(w.len);
  };
  auto advance = [&](DcWalk& w) {
    if (++w.c < w.units) return;
    w.c = 0;
    if (++w.grp < groups) return;
    w.grp = 0;
    if (++w.g < a.c.Hkv) return;
    w.g = 0;
    ++w.b;
    load_len(w);
  };
  DcWalk cw{sm.start[warp][0], sm.start[warp][1], sm.start[warp][2], sm.start[warp][3],
            sm.start[warp][4], sm.start[warp][5]};
  const int count = (int)(uq + (worker < ur ? 1 : 0));

  // ---- loads: chunk after chunk of this warp, the page numbers one ahead
  const int bs = min(a.c.page_shift, 5), br = 1 << bs;      // rows of a box of the 32 keys
  const int sub = lane & ((32 >> bs) - 1), dh = lane >> (5 - bs);
  const uint32_t ring = ptx::smem_u32(&sm.ring[warp * DC_SLOTS][0]);
  const uint32_t bar = ptx::smem_u32(&sm.full[warp * DC_SLOTS]);
  constexpr uint32_t SLOT = 32 * D * 2;
  DcWalk lw = cw;
  int ahead = 0;        // units that lw is past the first
  int is = 0;           // the slot to fill next
  int issued = 0;
  bool pend_v = false;  // the unit's K has been requested, its V is next
  int pend_page = 0, pend_row = 0, pend_head = 0;
  bool pend_mine = false, pend = false;
  auto look = [&] {     // the next unit with keys: its page number, not used yet
    pend = false;
    while (ahead < count) {
      const int base = lw.c * DC_UNIT;
      if (base < lw.len) {
        const int key = base + sub * br;
        pend_mine = dh < H2 && key < lw.len;
        if (pend_mine) pend_page = a.table[lw.b * a.table_stride + (key >> a.c.page_shift)];
        pend_row = key & ((1 << a.c.page_shift) - 1);
        pend_head = lw.g;
        pend = true;
        advance(lw);
        ++ahead;
        return;
      }
      advance(lw);
      ++ahead;
    }
  };
  auto issue = [&] {    // K or V of the unit looked up into the next slot
    if (!pend_v && pend_mine) pend_mine = pg_check(a.c, pend_page) >= 0;
    const uint32_t bytes = (uint32_t)__popc(__ballot_sync(0xffffffffu, pend_mine)) * br * 128u;
    if (lane == 0) ptx::mbar_arrive_expect_tx(bar + 8 * is, bytes + never);
    __syncwarp();
    if (pend_mine)
      ptx::tma_load_4d(ring + is * SLOT + (uint32_t)(dh * 4096 + sub * br * 128),
                       pend_v ? &tm_v : &tm_k, dh * 64, pend_row, pend_head, pend_page,
                       bar + 8 * is);
    is = is + 1 == DC_SLOTS ? 0 : is + 1;
    ++issued;
    if (pend_v) look();
    pend_v = !pend_v;
  };
  look();
  for (int i = 0; i < DC_SLOTS && pend; ++i) issue();

  // ---- compute
  const bool plain = a.cap == 0.f && a.slopes == nullptr && a.scale > 0.f;
  const float mul = plain ? a.scale * LOG2E : 1.f;
  uint32_t q[NB][D / 16][2];
  float m[NB][2], l[NB][2], slope[NB][2], o[D / 16][NB][4];
  // the queries of a segment, requested while the segment before it is joined
  auto load_q = [&](const DcWalk& w) {
    const int heads = min(16, G - w.grp * 16);
    const E* base = reinterpret_cast<const E*>(a.q) + w.b * a.q_ts + col2;
    const int first = w.g * G + w.grp * 16;
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
  bool whole = true;      // ... which begins in this warp
  int us = 0;             // the slot in use, and its phase
  uint32_t phase = 0;
  int used = 0;
  bool dead = false;
  // the slot's copy has landed / the slot is free: the next copy into it
  auto take = [&] {
    dead = !__all_sync(0xffffffffu, ptx::mbar_wait(bar + 8 * us, phase, tmo, &sm.abort_flag));
  };
  auto give = [&] {
    __syncwarp();
    ++used;
    us = us + 1 == DC_SLOTS ? 0 : us + 1;
    if (us == 0) phase ^= 1u;
    if (pend) {
      ptx::fence_proxy_async_smem();
      issue();
    }
  };
  // shared-memory offsets of this lane's matrix rows: 16 of K, 8 + 8 of V
  uint32_t ko[4], vo[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    ko[e] = dc_swz(lane & 15, 2 * e + (lane >> 4));
    vo[e] = dc_swz((lane & 7) + 8 * (lane >> 4), 2 * e + ((lane >> 3) & 1));
  }
  // Scores of a unit capped and biased, in log2 units; the query is `ahead` of its
  // first key.
  auto score = [&](float (&sc)[2][NB][4], int ahead) {
    auto each = [&](auto f) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int nbk = 0; nbk < NB; ++nbk)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            f(sc[mt][nbk][i], slope[nbk][i & 1], 16 * mt + row4 + 8 * (i >> 1));
    };
    const float kk = a.scale * LOG2E;
    if (a.cap > 0.f) {
      const float A = a.cap * LOG2E, ratio = pg_cap_ratio(a.scale, a.cap);
      bool large = false;
      each([&](float& v, float, int) { large |= !(fabsf(v * ratio) <= 0.5f); });
      large = __any_sync(0xffffffffu, large);
      each([&](float& v, float, int) { v = pg_capped(v, kk, ratio, A, large); });
    } else {
      each([&](float& v, float, int) { v *= kk; });
    }
    each([&](float& v, float sl, int key) { v = fmaf(-sl, (float)(ahead - key), v); });
  };
  for (int u = 0; u < count; ++u) {
    const int h0 = cw.g * G + cw.grp * 16;  // first query head
    const int heads = min(16, G - cw.grp * 16);
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
    const int base = cw.c * DC_UNIT;
    const int have = min(32, cw.len - base);
    if (have > 0 && !dead) {
      take();
      if (!dead) {
        const uint32_t ks = ring + us * SLOT;
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
            dc_ldsm(ks + (e >> 2) * 4096 + mt * 2048 + ko[e & 3], r);
#pragma unroll
            for (int nbk = 0; nbk < NB; ++nbk)
              dc_mma<E>(sc[mt][nbk], r, q[nbk][e][0], q[nbk][e][1]);
          }
        }
        give();
        if (!plain) score(sc, cw.len - 1 - base);
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
        // P^T of 16 keys: B fragments.  A weight goes to the sum in two parts, rounded and
        // the rest (22 or 16 bits of it), as the dense cache's kernel for 64-wide heads
        // passes it on: the tensor pipe is idle nine tenths of the time here.
        uint32_t pb[2][NB][2], pl[2][NB][2];
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
            const uint32_t h0 = Ty::pack(p0, p1), h1 = Ty::pack(p2, p3);
            const float2 f0 = Ty::to_f2(h0), f1 = Ty::to_f2(h1);
            pb[mt][nbk][0] = dc_transpose(h0);
            pb[mt][nbk][1] = dc_transpose(h1);
            pl[mt][nbk][0] = dc_transpose(Ty::pack(p0 - f0.x, p1 - f0.y));
            pl[mt][nbk][1] = dc_transpose(Ty::pack(p2 - f1.x, p3 - f1.y));
          }
        take();
        if (!dead) {
          const uint32_t vs = ring + us * SLOT;
          if (have < 32) {  // rows behind the last key may hold anything: 0 x NaN is NaN
            uint8_t* vr = &sm.ring[warp * DC_SLOTS + us][0];
            for (int x = have * 8 + lane; x < 32 * 8; x += 32)
#pragma unroll
              for (int hb = 0; hb < H2; ++hb)
                *reinterpret_cast<uint4*>(vr + hb * 4096 + x * 16) = make_uint4(0u, 0u, 0u, 0u);
            __syncwarp();
          }
          // O^T: dims 16 e + row4 (+ 8), heads col2 (+ 1)
#pragma unroll
          for (int e = 0; e < D / 16; ++e)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
              uint32_t r[4];
              dc_ldsm_t(vs + (e >> 2) * 4096 + mt * 2048 + vo[e & 3], r);
#pragma unroll
              for (int nbk = 0; nbk < NB; ++nbk)
                dc_mma<E>(o[e][nbk], r, pb[mt][nbk][0], pb[mt][nbk][1]);
#pragma unroll
              for (int nbk = 0; nbk < NB; ++nbk)
                dc_mma<E>(o[e][nbk], r, pl[mt][nbk][0], pl[mt][nbk][1]);
            }
          give();
        }
      }
    }

    const DcWalk now = cw;
    advance(cw);
    if (cw.c != 0 && u + 1 < count) continue;
    // ---- the end of this warp's part of the segment
    fresh = true;
    if (u + 1 < count) load_q(cw);
    const bool done = now.c == now.units - 1;     // the part has the segment's last unit
    const bool full = whole && done;
    if (lane == 0) {
      int2* info = side.seg + (int64_t)now.b * segs + now.g * groups + now.grp;
      if (whole) info->x = worker;
      if (done) info->y = worker;
    }
    const int slot = 2 * worker + (whole ? 1 : 0);
    // where head h of the group goes, if not to the output: row of parts or side
    auto part_row = [&](int h) {
      return full ? (int64_t)(parts.count - 1) * parts.rows + (int64_t)now.b * a.Hq + h0 + h
                  : (int64_t)slot * 16 + h;
    };
    float* const po = full ? parts.o : side.o;
    float* const pl = full ? parts.lse : side.lse;
    const bool direct = full && !prefix;
#pragma unroll
    for (int nbk = 0; nbk < NB; ++nbk) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float v = l[nbk][x];
#pragma unroll
        for (int sh = 4; sh < 32; sh <<= 1) v += __shfl_xor_sync(0xffffffffu, v, sh);
        const float inv = v == 0.f ? 0.f : 1.f / v;  // no keys: 0; a NaN goes on
        const int h = 8 * nbk + col2 + x;
        if (row4 == 0 && h < heads && !direct)
          pl[part_row(h)] = v == 0.f ? -INFINITY : m[nbk][x] + log2f(v);
#pragma unroll
        for (int e = 0; e < D / 16; ++e) {
          const int r = Sm::HEADS == 8 ? col2 + x : lane & 3;
          sm.out[warp][r][16 * e + row4] = o[e][nbk][x] * inv;
          sm.out[warp][r][16 * e + row4 + 8] = o[e][nbk][2 + x] * inv;
        }
        if (Sm::HEADS == 8 && x == 0) continue;
        __syncwarp();
        for (int i = lane; i < Sm::HEADS * (D / 8); i += 32) {
          const int hr = i / (D / 8), d = 8 * (i % (D / 8));
          const int h = 8 * nbk + (Sm::HEADS == 8 ? hr : 2 * hr + x);
          if (h >= heads) break;
          const float4 v = *reinterpret_cast<const float4*>(&sm.out[warp][hr][d]);
          const float4 w = *reinterpret_cast<const float4*>(&sm.out[warp][hr][d + 4]);
          if (direct) {
            *reinterpret_cast<uint4*>(reinterpret_cast<E*>(a.out) + now.b * a.o_ts +
                                      (int64_t)(h0 + h) * a.o_hs + d) =
                make_uint4(Ty::pack(v.x, v.y), Ty::pack(v.z, v.w), Ty::pack(w.x, w.y),
                           Ty::pack(w.z, w.w));
          } else {
            float* dst = po + part_row(h) * D + d;
            *reinterpret_cast<float4*>(dst) = v;
            *reinterpret_cast<float4*>(dst + 4) = w;
          }
        }
        __syncwarp();  // sm.out is free again
      }
    }
  }
  if (dead) {         // copies in flight land before the shared memory goes
    for (int k = used; k < issued; ++k) {
      const long long t0 = clock64();
      while (!ptx::mbar_try_wait(bar + 8 * (k % DC_SLOTS), (uint32_t)(k / DC_SLOTS) & 1u))
        if (clock64() - t0 > (long long)(tmo * 2ull)) break;
    }
    if (lane == 0) pg_error(a.c, DDQ_ERR_TIMEOUT);
  }
  if (prefix) ptx::pdl_wait();
}

// Joins the parts of every row, in order: the prefix splits, then the own keys
// (whole, or the side slots of the warps that share them).
//   o = sum_z 2^(lse_z - max) o_z / sum_z 2^(lse_z - max)
// One warp per row, or, with few rows (of long sequences: many parts), eight.
template <typename E, int D, int WPR>
__global__ void __launch_bounds__(256)
    paged_decode_merge_kernel(const PgAttnArgs a, const PgParts p, const DcSide side) {
  using Ty = PgType<E>;
  constexpr int DPL = D / 32;
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int64_t row = WPR == 1 ? (int64_t)blockIdx.x * 8 + warp : blockIdx.x;
  if (row >= (int64_t)a.T * a.Hq) return;
  const int b = (int)((uint32_t)row / (uint32_t)a.Hq), h = (int)row - b * a.Hq;  // rows < 2^31
  const int G = a.G, groups = dc_groups(G);
  const int g = h / G, hh = h - g * G;
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
    for (int z1 = WPR == 1 ? 0 : 4 * warp; z1 < m; z1 += 4 * WPR) {  // four in flight
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
  if constexpr (WPR > 1) {
    __shared__ float so[WPR][D], sd[WPR];
#pragma unroll
    for (int e = 0; e < DPL; ++e) so[warp][lane * DPL + e] = o[e];
    if (lane == 0) sd[warp] = den;
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int w = 1; w < WPR; ++w) {
      den += sd[w];
#pragma unroll
      for (int e = 0; e < DPL; ++e) o[e] += so[w][lane * DPL + e];
    }
  }
  const float inv = den == 0.f ? 0.f : 1.f / den;  // NaN stays NaN
  E* dst = reinterpret_cast<E*>(a.out) + b * a.o_ts + (int64_t)h * a.o_hs + lane * DPL;
#pragma unroll
  for (int e = 0; e < DPL; e += 2)
    *reinterpret_cast<uint32_t*>(dst + e) = Ty::pack(o[e] * inv, o[e + 1] * inv);
}

template <int D>
constexpr int dc_smem_bytes() { return (int)sizeof(DcSmem<D>) + 1024; }
// an SM has 228 KB for its CTAs, 1 KB of each CTA's its own
static_assert(dc_resident(64, 1) * (dc_smem_bytes<64>() + 1024) <= 228 * 1024, "resident CTAs");
static_assert(dc_resident(128, 1) * (dc_smem_bytes<128>() + 1024) <= 228 * 1024, "resident CTAs");

// CTAs that fit the GPU at once.
int dc_ctas(int64_t B, int Hq, int Hkv, int D, int64_t keys, int sms) {
  const int64_t units = B * Hkv * dc_groups(Hq / Hkv) * ((keys + DC_UNIT - 1) / DC_UNIT);
  const int64_t most = (units + DC_NW - 1) / DC_NW;
  const int64_t fit = (int64_t)sms * dc_resident(D, Hq / Hkv > 8 ? 2 : 1);
  return (int)(most < 1 ? 1 : most < fit ? most : fit);
}

DcPlan dc_plan(int64_t B, int Hq, int Hkv, int D, int64_t keys, int64_t prefix, int sms) {
  DcPlan p;
  p.ctas = dc_ctas(B, Hq, Hkv, D, keys, sms);
  p.splits = prefix ? tc_splits(B, 1, Hq, Hkv, prefix, false, sms) : 0;
  const int64_t rows = B * Hq, count = prefix ? p.splits + 1 : 0;
  p.off_lse = (size_t)count * rows * D * 4;
  p.off_so = p.off_lse + ((size_t)count * rows * 4 + 15) / 16 * 16;
  p.off_sl = p.off_so + (size_t)p.ctas * DC_NW * 2 * 16 * D * 4;
  p.off_seg = p.off_sl + (size_t)p.ctas * DC_NW * 2 * 16 * 4;
  p.bytes = p.off_seg + (size_t)B * Hkv * dc_groups(Hq / Hkv) * sizeof(int2);
  return p;
}

int launch_paged_decode(const PgAttnArgs& a, bool bf16, void* ws, const DcPlan& plan,
                        unsigned long long tmo, int debug_flags, cudaStream_t s) {
  if (a.R > DC_MAXB) return DDQ_ERR_SHAPE;
  uint8_t* w = static_cast<uint8_t*>(ws);
  const int count = a.prefix_len ? plan.splits + 1 : 0;
  const PgParts parts{count ? reinterpret_cast<float*>(w) : nullptr,
                      count ? reinterpret_cast<float*>(w + plan.off_lse) : nullptr,
                      (int64_t)a.T * a.Hq, count};
  const DcSide side{reinterpret_cast<float*>(w + plan.off_so),
                    reinterpret_cast<float*>(w + plan.off_sl),
                    reinterpret_cast<int2*>(w + plan.off_seg)};
  int st = DDQ_OK;
  if (count) {
    st = launch_paged_tc(a, bf16, parts, plan.splits, tmo, debug_flags, s);
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
    // test hook (ddq_set_debug bit 0): 16 bytes that never come, so that the warps'
    // bounded waits run out and they wind down
    e = cudaLaunchKernelEx(&cfg, kern, tk, tv, a, parts, side, tmo, 16 * (debug_flags & 1));
    return DDQ_OK;
  };
  const bool wide = a.Hq / a.c.Hkv > 8;
#define DDQ_DC(D_, NB_)                                                                        \
  (bf16 ? go(paged_decode_kernel<__nv_bfloat16, D_, NB_>, attr[1][D_ / 128][NB_ - 1],          \
             dc_smem_bytes<D_>())                                                         \
        : go(paged_decode_kernel<__half, D_, NB_>, attr[0][D_ / 128][NB_ - 1],                 \
             dc_smem_bytes<D_>()))
  if (a.c.D == 64)
    st = wide ? DDQ_DC(64, 2) : DDQ_DC(64, 1);
  else
    st = wide ? DDQ_DC(128, 2) : DDQ_DC(128, 1);
#undef DDQ_DC
  if (st) return st;
  if (e == cudaSuccess) {
    const int64_t rows = (int64_t)a.T * a.Hq;
    const bool few = rows <= 16 * (int64_t)device_sm_count(dev);
    cfg.gridDim = dim3((unsigned)(few ? rows : (rows + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
#define DDQ_DM(E_, D_)                                                                        \
  (few ? cudaLaunchKernelEx(&cfg, paged_decode_merge_kernel<E_, D_, 8>, a, parts, side)       \
       : cudaLaunchKernelEx(&cfg, paged_decode_merge_kernel<E_, D_, 1>, a, parts, side))
    if (bf16)
      e = a.c.D == 64 ? DDQ_DM(__nv_bfloat16, 64) : DDQ_DM(__nv_bfloat16, 128);
    else
      e = a.c.D == 64 ? DDQ_DM(__half, 64) : DDQ_DM(__half, 128);
#undef DDQ_DM
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return DDQ_ERR_LAUNCH;
  }
  return check_launch();
}

}  // namespace ddq
