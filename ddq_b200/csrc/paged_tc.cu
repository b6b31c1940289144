// paged_tc.cu - paged attention of many query rows on the tcgen05 tensor cores:
// the new tokens of ragged requests, and the rows of a decode batch over the
// prefix that they share.
//
// Row (t, h), key head g = h / (Hq / Hkv), at position p, attends the keys j of
// its own request (and of the shared prefix, which comes first) with j < end:
//   s_j = scale q . k_j          (capped: cap * tanh(s_j / cap))
//   z_j = s_j - slope_h |p - j|
//   o   = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m),   m = max_j z_j
// and o = 0 where there is no such key.  A prompt's row has
// end = max(p + 1, prefix_len + min(bidir, len)), a decode row all keys.
//
// The G = Hq / Hkv query heads of a key/value head are packed with the tokens:
// row rr of a request is token rr / G, head g G + rr % G, so that a tile of 256
// rows covers 256 / G consecutive tokens, every key tile is used by all heads
// that share it, and few tokens still fill a tile (a decode batch of B rows is
// a request of B tokens).
//
// One CTA per (tile, key/value head, split of the key axis), two 128-row
// halves, one key tile of 128 at a time:
//   S_t = Q_t K^T   tcgen05.mma, 128 x 128, from shared memory into TMEM
//   P_t = exp2(x - m) of the scores x in log2 units, one thread per row, fp32;
//         rounded once to the operand type (weights reach PV in 11 or 8 bits,
//         the sum l is of the unrounded ones) and put back into TMEM
//   O_t += P_t V    tcgen05.mma, A from TMEM, V from shared memory as it lies
//         (keys in rows: an MN-major B operand, no transpose)
// The running maximum only moves when a tile exceeds it by more than 8 (a
// factor 256, harmless in fp32 and in the type of P), so O in TMEM is rarely
// rescaled: after the first tiles a row's maximum hardly grows.
//
// Warps 0-3 and 4-7: softmax of half 0 and 1.  Warp 8: TMA, one box per page
// and 64 dimensions, each lane its own.  Warps 9 and 10: MMA issue, a half each.
// S, one for both halves in turn, is free as soon as its rows are in registers, so
// the next scores are made during the softmax, and the halves stay half a tile
// apart: while one uses the special-function pipe, the other loads and stores (with
// an S each they ran in step: 97.7 us instead of 93.0 for 509 tokens behind 32259
// keys, 64-wide heads).
#include <cudaTypedefs.h>

#include <mutex>
#include <type_traits>

#include "launch.cuh"
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace ddq {

constexpr int TC_KV = 128;       // keys per tile
constexpr int TC_HALF = 128;     // rows per half
constexpr int TC_ROWS = 256;     // rows per CTA
constexpr int TC_NT = 384;        // two softmax warpgroups and one for TMA and MMA issue
// Registers a thread: launched with 168 (3 warps on each quarter of the SM);
// the third warpgroup gives up 80, the softmax ones take 40 each: 256 x 208 +
// 128 x 88 = 384 x 168.  A softmax thread holds its row of 128 scores (the plain
// kernels spill 16 bytes at that, the scored ones nothing).
constexpr int TC_REG_SOFTMAX = 208, TC_REG_ISSUE = 88;
constexpr float TC_LAZY = 8.f;   // log2 units

template <int D>
struct TcLayout {
  static constexpr int HB = TC_KV * 128;         // bytes of 128 rows x 64 elements
  static constexpr int TILE = (D / 64) * HB;     // one K or V tile, one half of Q
  static constexpr int ST = D == 64 ? 8 : 4;     // ring stages (K and V alternate)
  static constexpr int OFF_RING = 2 * TILE;
  static constexpr int OFF_BAR = OFF_RING + ST * TILE;
  static constexpr int SMEM = OFF_BAR + 512 + 1024;
  // TMEM columns: scores (of both halves in turn), weights and outputs of each half
  static constexpr int COL_S = 0, COL_P = 128, COL_O = 256;
};

__device__ __forceinline__ float tc_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void tc_sts(uint32_t p, uint32_t a, uint32_t b, uint32_t c,
                                       uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(p), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}

__device__ __forceinline__ uint4 tc_lds(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(p)
               : "memory");
  return v;
}

__device__ __forceinline__ void tc_regs(uint32_t* r) {  // the loads above are complete
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    asm volatile(""
                 : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]),
                   "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}

// Two fp32 values in a register pair and the packed operations on them (half the
// issue slots).
struct TcF2 {
  uint64_t v;
};
__device__ __forceinline__ TcF2 tc_pk(float a, float b) {
  TcF2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ TcF2 tc_pk1(float a) { return tc_pk(a, a); }
__device__ __forceinline__ void tc_un(TcF2 x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v));
}
__device__ __forceinline__ TcF2 tc_fma2(TcF2 a, TcF2 b, TcF2 c) {
  TcF2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ TcF2 tc_mul2(TcF2 a, TcF2 b) {
  TcF2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ TcF2 tc_add2(TcF2 a, TcF2 b) {
  TcF2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// 2^x for x <= 8 on the FMA pipe: x = n + f with n the nearest integer (adding
// 1.5 2^23 leaves it in the low bits), 2^f by the minimax polynomial of degree 4
// on [-1/2, 1/2] (Remez, relative error 2^-18.5: 2^-7 of the rounding of a
// weight to 11 bits), n added to the exponent field.  Below 2^-126: 2^-126.
__device__ __forceinline__ TcF2 tc_poly_exp2(float x0, float x1) {
  constexpr float M = 12582912.f;
  const TcF2 x = tc_pk(fmaxf(x0, -126.f), fmaxf(x1, -126.f));
  const TcF2 t = tc_add2(x, tc_pk(M, M));
  const TcF2 f = tc_add2(x, tc_mul2(tc_add2(t, tc_pk(-M, -M)), tc_pk(-1.f, -1.f)));
  TcF2 p = tc_fma2(f, tc_pk(0x1.3997d6p-7f, 0x1.3997d6p-7f), tc_pk(0x1.ca1440p-5f, 0x1.ca1440p-5f));
  p = tc_fma2(p, f, tc_pk(0x1.ec06dap-3f, 0x1.ec06dap-3f));
  p = tc_fma2(p, f, tc_pk(0x1.62e0dcp-1f, 0x1.62e0dcp-1f));
  p = tc_fma2(p, f, tc_pk(0x1.ffffe8p-1f, 0x1.ffffe8p-1f));
  float p0, p1, t0, t1;
  tc_un(p, p0, p1);
  tc_un(t, t0, t1);
  return tc_pk(__uint_as_float(__float_as_uint(p0) + (__float_as_uint(t0) << 23)),
               __uint_as_float(__float_as_uint(p1) + (__float_as_uint(t1) << 23)));
}

// Wait for a phase of a barrier, bounded like ptx::mbar_wait, but the caller goes
// on in either case: after a wait that gave up (abort set, DDQ_ERR_TIMEOUT at the
// end) every later one returns at once, the loops run out on whatever the
// buffers hold, and no lane leaves its warp in between.  A wait on a phase that
// is complete costs 55 cycles this way; with an answer for the warp to branch on
// it cost 106, six times per pair of tiles on the path from P to the next S.
__device__ __forceinline__ void tc_wait(uint32_t bar, uint32_t parity, uint64_t tmo,
                                        volatile int* abort) {
  if (!ptx::mbar_try_wait_now(bar, parity)) {
    const long long t0 = clock64();
    while (!ptx::mbar_try_wait(bar, parity)) {
      if (*abort || clock64() - t0 > (long long)(tmo * 2ull)) {
        *abort = 1;
        break;
      }
    }
  }
  __syncwarp();
}

// One arrival for the warp, after all its lanes got here.
__device__ __forceinline__ void tc_arrive(uint32_t bar, int lane) {
  __syncwarp();
  if (lane == 0) ptx::mbar_arrive(bar);
}

__device__ __forceinline__ float tc_max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// SCORED: scores that are capped or biased, or whose scale is not positive; the
// plain kernel has none of that code.
template <typename E, int D, bool SCORED>
__global__ void __launch_bounds__(TC_NT, 1)
    paged_tc_kernel(const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v, const PgAttnArgs a,
                    const PgParts parts, const int splits, const int skip_signal,
                    const unsigned long long tmo) {
  using L = TcLayout<D>;
  using Ty = PgType<E>;
  extern __shared__ uint8_t tc_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tc_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const uint32_t sbase = ptx::smem_u32(smem);
  __shared__ int found[6], wsum[TC_NT / 32];  // request, tile, first row, rows, keys, bidir
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tile0 = (int)(blockIdx.x / (unsigned)a.c.Hkv);
  const int G = a.G, g = (int)blockIdx.x - tile0 * a.c.Hkv, z = blockIdx.y;

  const uint32_t bar_full = sbase + L::OFF_BAR;
  const uint32_t bar_empty = bar_full + 8 * L::ST;
  const uint32_t bar_q = bar_empty + 8 * L::ST;
  const uint32_t bar_s = bar_q + 8;         // [2] scores ready
  const uint32_t bar_sfree = bar_s + 16;    // [2] scores read
  const uint32_t bar_p = bar_sfree + 16;    // [2] weights ready
  const uint32_t bar_p2 = bar_p + 16;       // [2] ... of the tile's second 64 keys
  const uint32_t bar_pv = bar_p2 + 16;      // [2] PV done
  const uint32_t bar_drain = bar_pv + 16;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::OFF_BAR + 8 * (2 * L::ST + 13));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  if (tid == 0) {
    for (int s = 0; s < L::ST; ++s) {
      ptx::mbar_init(bar_full + 8 * s, 1);
      ptx::mbar_init(bar_empty + 8 * s, 2);  // the MMAs of both halves
    }
    ptx::mbar_init(bar_q, 8);  // warps
    for (int t = 0; t < 2; ++t) {
      ptx::mbar_init(bar_s + 8 * t, 1);
      ptx::mbar_init(bar_sfree + 8 * t, 4);
      ptx::mbar_init(bar_p + 8 * t, 4);
      ptx::mbar_init(bar_p2 + 8 * t, 4);
      ptx::mbar_init(bar_pv + 8 * t, 1);
    }
    ptx::mbar_init(bar_drain, 1);
    ptx::mbar_init(bar_drain + 8, 1);
    *abort_flag = 0;
    found[0] = -1;
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tm_k);
    ptx::prefetch_tmap(&tm_v);
  }
  if (warp == 9) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_holder), 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();

  // ---- the request and the tile of this CTA, kv heads next to each other: the CTAs
  // that start last shall have the fewest keys, so the tiles of a request go from the
  // last to the first and of up to 32 requests the longest is first (7679 tokens of 12
  // documents: in the order of the batch 8 us more, a head after the other 34; four
  // prompts of 4096 tokens, 486 us: a head after the other 10)
  int r = 0, tile = tile0, t_first = 0, n = a.T;
  int len = 0, most = 0;  // own keys, and the ones that bidir lets every row attend
  if (a.cu && a.R <= 32) {  // each warp for itself: one round of loads, no barrier
    const int rr = a.R - 1 - lane;
    int c0 = 0, cn = 0, ln = 0, bd = 0;
    if (rr >= 0) {
      c0 = a.cu[rr];
      cn = a.cu[rr + 1] - c0;
      ln = a.lens[rr];
      if (a.bidir) bd = a.bidir[rr];
      if (c0 < 0 || c0 >= a.T || cn < 0) c0 = cn = 0;
    }
    const int tiles = (min(cn, a.T - c0) * G + TC_ROWS - 1) / TC_ROWS;
    int s = 0;
#pragma unroll 4
    for (int e = 0; e < a.R; ++e) {
      const int le = __shfl_sync(0xffffffffu, ln, e), te = __shfl_sync(0xffffffffu, tiles, e);
      if (le > ln || (le == ln && e <= lane)) s += te;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, tile < s && tile >= s - tiles);
    if (hit == 0) {  // the grid covers the most tiles that T rows can make
      if (warp == 9) ptx::tmem_dealloc(*tmem_holder, 512);
      return;
    }
    const int src = __ffs(hit) - 1;
    r = __shfl_sync(0xffffffffu, rr, src);
    tile = __shfl_sync(0xffffffffu, s, src) - 1 - tile;
    t_first = __shfl_sync(0xffffffffu, c0, src);
    n = __shfl_sync(0xffffffffu, cn, src);
    len = pg_clamp_len(a, __shfl_sync(0xffffffffu, ln, src));
    most = __shfl_sync(0xffffffffu, bd, src);
  } else if (a.cu) {
    int run = 0;
    for (int base = 0; base < a.R; base += TC_NT) {
      const int rr = a.R - 1 - (base + tid);
      int c0 = 0, cn = 0, ln = 0, bd = 0;
      if (rr >= 0) {  // one round of loads; the CTA's request is among them
        c0 = a.cu[rr];
        cn = a.cu[rr + 1] - c0;
        ln = a.lens[rr];
        if (a.bidir) bd = a.bidir[rr];
        if (c0 < 0 || c0 >= a.T || cn < 0) c0 = cn = 0;
      }
      const int tiles = (min(cn, a.T - c0) * G + TC_ROWS - 1) / TC_ROWS;
      int s = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
      }
      if (lane == 31) wsum[warp] = s;
      __syncthreads();
      int before = run;
      for (int w = 0; w < TC_NT / 32; ++w) {
        const int x = wsum[w];
        if (w < warp) before += x;
        run += x;
      }
      s += before;
      if (tile < s && tile >= s - tiles) {
        found[0] = rr;
        found[1] = s - 1 - tile;
        found[2] = c0;
        found[3] = cn;
        found[4] = pg_clamp_len(a, ln);
        found[5] = bd;
      }
      __syncthreads();
      if (found[0] >= 0) break;
    }
    r = found[0];
    if (r < 0) {
      if (warp == 9) ptx::tmem_dealloc(*tmem_holder, 512);
      return;
    }
    tile = found[1];
    t_first = found[2];
    n = found[3];
    len = found[4];
    most = found[5];
  }
  const int P = a.prefix_len;
  const int least = a.cu ? (a.bidir ? P + min(most, len) : 0) : P;
  // n new tokens, the last of them without a row where q ends before cu does: the rows
  // that exist keep their positions
  const int row0 = tile * TC_ROWS, nrow = min(TC_ROWS, min(n, a.T - t_first) * G - row0);
  const int halves = nrow > TC_HALF ? 2 : 1;
  // keys of the row of token i: those below end(i); the last row has the most
  auto end_of = [&](int i) {
    const int e = a.cu ? P + len - n + i + 1 : 0;
    return max(max(e, least), 0);
  };
  const int end_max = end_of((row0 + nrow - 1) / G);
  const int np = (min(P, end_max) + TC_KV - 1) / TC_KV;
  const int nt = np + (max(end_max - P, 0) + TC_KV - 1) / TC_KV;
  int lo = 0, cnt = nt;
  if (splits > 1) {  // (below 2^24 tiles in at most 64 parts)
    lo = (int)((uint32_t)nt * (uint32_t)z / (uint32_t)splits);
    cnt = (int)((uint32_t)nt * (uint32_t)(z + 1) / (uint32_t)splits) - lo;
  }
  // tile k of this CTA: first key, keys that exist behind it, its list
  auto key0 = [&](int k) { return lo + k < np ? (lo + k) * TC_KV : P + (lo + k - np) * TC_KV; };
  auto limit = [&](int k) { return lo + k < np ? P : P + len; };

  if (cnt == 0) {  // no keys: zeros, or an empty part
    if (tid < nrow) {
      const int tok = t_first + (row0 + tid) / G, h = g * G + (row0 + tid) % G;
      if (parts.o) {
        parts.lse[(int64_t)z * parts.rows + (int64_t)tok * a.Hq + h] = -INFINITY;
      } else {
        E* dst = reinterpret_cast<E*>(a.out) + tok * a.o_ts + (int64_t)h * a.o_hs;
#pragma unroll
        for (int c = 0; c < D; c += 8)
          *reinterpret_cast<uint4*>(dst + c) = make_uint4(0u, 0u, 0u, 0u);
      }
    }
    if (warp == 9) ptx::tmem_dealloc(*tmem_holder, 512);
    return;
  }

  const uint32_t tmem = *tmem_holder;

  if (warp < 8) {
    ptx::reg_inc<TC_REG_SOFTMAX>();
    // ---------------------------------------------------------------- softmax
    const int t = warp >> 2;
    const int rr = row0 + tid;                  // tid < 256: both halves in order
    const bool real = tid < nrow;
    const int i = real ? (int)((unsigned)rr / (unsigned)G) : 0, h = g * G + (real ? rr - i * G : 0);
    const int tok = t_first + i;
    // a row behind the last takes part unmasked (its Q is zero, its result is not
    // stored): a warp of such rows has no slower tiles than the others
    const int end = real ? end_of(i) : 0x7fffffff;
    const int pos = a.cu ? P + len - n + i : P + pg_len(a, real ? tok : 0) - 1;
    // A row's own key, at distance 0, keeps its final maximum above -cap: starting
    // there, keys far off under a steep bias come out as zeros at once and do not
    // raise the maximum tile by tile, rescaling O.
    float m = SCORED && a.cap > 0.f && pos >= 0 ? -a.cap * 1.4426950408889634f : -INFINITY;
    float l = 0.f;
    const bool half_on = t < halves;
    // This warp's 32 rows of Q, K-major with the 128-byte swizzle, and later its
    // rows of the output, through the same shared memory (Q is done with when the
    // last scores are there): D / 8 lanes read or write a row together, all pieces in
    // flight at once (loads into registers came back one after another: 9 thousand
    // cycles instead of 3 for 256 rows of 128 elements).
    uint8_t* const rows = smem + t * L::TILE + (warp & 3) * 32 * 128;
    auto piece = [&](int row, int c) {  // 16-byte piece c of 64-element block 0
      return row * 128 + ((c ^ (row & 7)) << 4);
    };
    {
      const int64_t q_off = real ? tok * a.q_ts + (int64_t)h * a.q_hs : -1;
      constexpr int LPR = D / 8;  // lanes per row
#pragma unroll
      for (int e = 0; e < LPR; ++e) {
        const int64_t off = __shfl_sync(0xffffffffu, q_off, e * (32 / LPR) + lane / LPR);
        const int row = e * (32 / LPR) + lane / LPR, c = lane % LPR;
        const E* src = reinterpret_cast<const E*>(a.q) + (off >= 0 ? off : 0) + 8 * c;
        ptx::cp_async16_zfill(ptx::smem_u32(rows + (c >> 3) * L::HB + piece(row, c & 7)), src,
                              off >= 0);
      }
      ptx::cp_async_wait_all();
      ptx::fence_proxy_async_smem();
      tc_arrive(bar_q, lane);
    }
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + L::COL_S + lanes;
    const uint32_t tp = tmem + L::COL_P + t * 64 + lanes;
    const uint32_t to = tmem + L::COL_O + t * D + lanes;
    if (half_on) {
      constexpr float LOG2E = 1.4426950408889634f;
      const float kk = a.scale * LOG2E, mul = SCORED ? 1.f : kk;
      const float slope = SCORED && a.slopes ? a.slopes[h] * LOG2E : 0.f;
      const float r2 = SCORED && a.cap > 0.f ? (a.scale / a.cap) * (a.scale / a.cap) : 0.f;
      const float r8 = (r2 * r2) * (r2 * r2);
      const TcF2 cap0 = tc_pk1(a.cap > 0.f ? kk * PG_TANH0 : kk),
                 cap1 = tc_pk1(kk * PG_TANH1 * r2),
                 cap2 = tc_pk1(kk * PG_TANH2 * (r2 * r2)),
                 cap3 = tc_pk1(kk * PG_TANH3 * (r2 * r2 * r2)),
                 cap4 = tc_pk1(kk * PG_TANH4 * r8);
      // |y| <= 1/2, y = scale s / cap: cap tanh(y) = scale s P(y^2), the coefficients in
      // powers of s^2; up to |y| = 1/6 the minimax polynomial of degree 2 (error
      // 2^-24.7): six or four packed operations for two scores, their bias added, and no
      // special function.  Without a cap P is 1.
      auto capped_poly = [&](TcF2 x) {
        const TcF2 v = tc_mul2(x, x);
        return tc_fma2(v, tc_fma2(v, tc_fma2(v, tc_fma2(v, cap4, cap3), cap2), cap1), cap0);
      };
      auto capped = [&](float s0, float s1) {
        const TcF2 x = tc_pk(s0, s1);
        return tc_mul2(x, capped_poly(x));
      };
      auto capped_add = [&](float s0, float s1, TcF2 b) {
        const TcF2 x = tc_pk(s0, s1);
        return tc_fma2(x, capped_poly(x), b);
      };
      // the largest scores for the polynomials; their powers and coefficients are finite
      const float poly_max = !(kk * r8 < 1e30f && kk * r8 > -1e30f) ? -1.f
                             : a.cap > 0.f ? fminf(0.5f * a.cap / fabsf(a.scale), 1e18f)
                                           : 1e18f;
      const TcF2 low0 = tc_pk1(a.cap > 0.f ? kk * 0.999999965f : kk),
                 low1 = tc_pk1(kk * -0.333310343f * r2),
                 low2 = tc_pk1(kk * 0.131114860f * (r2 * r2));
      const float poly2_max = a.cap > 0.f ? poly_max * (1.f / 3) : poly_max;
      for (int k = 0; k < cnt; ++k) {
        const int j0 = key0(k);
        const int lim = min(end, limit(k)) - j0;  // keys of this tile that the row attends
        const bool full = __all_sync(0xffffffffu, lim >= TC_KV);
        tc_wait(bar_s + 8 * t, (uint32_t)k & 1u, tmo, abort_flag);
        ptx::tc_fence_after();
        // the row into registers, and S is free for the next scores
        uint32_t u[128];
        float* s = reinterpret_cast<float*>(u);
        auto load_row = [&]() {
#pragma unroll
          for (int c = 0; c < 128; c += 32) ptx::tmem_ld_32x32b_x32(ts + c, u + c);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 128; c += 32) tc_regs(u + c);
        };
        load_row();
        bool poly = false;
        float step = 0.f, big = 0.f;
        if constexpr (SCORED) {
          // to log2 units, capped and biased.  Where the polynomial serves all scores of
          // the warp: in registers, below.  Otherwise 32 scores at a time and back to S,
          // so that this rarer code, with more of its values alive, does not take
          // registers from the rest (all in registers it spilled: 22 us more
          // for 7679 tokens of 12 packed documents, 128-wide heads).
          const float d0 = (float)(pos - j0);
          big = 0.f;
#pragma unroll
          for (int c = 0; c < 128; c += 2) big = tc_max3(big, fabsf(s[c]), fabsf(s[c + 1]));
          poly = __all_sync(0xffffffffu, big <= poly_max);
          if (!poly) {
            const float ratio = a.cap > 0.f ? pg_cap_ratio(a.scale, a.cap) : 0.f;
            const float A = a.cap * LOG2E;
#pragma unroll 1
            for (int c0 = 0; c0 < TC_KV; c0 += 32) {
              uint32_t o[32];
              ptx::tmem_ld_32x32b_x32(ts + c0, o);
              ptx::tmem_ld_wait();
              tc_regs(o);
              float* x = reinterpret_cast<float*>(o);
              const float dc = d0 - (float)c0;
              if (a.cap > 0.f) {  // each score by its own size: rows of small ones
                // beside one above half the cap keep their value
#pragma unroll
                for (int c = 0; c < 32; ++c) x[c] = pg_capped(x[c], kk, ratio, A, true);
              } else {
#pragma unroll
                for (int c = 0; c < 32; ++c) x[c] *= kk;
              }
              if (a.slopes) {
#pragma unroll
                for (int c = 0; c < 32; ++c) x[c] = fmaf(-slope, fabsf(dc - (float)c), x[c]);
              }
              ptx::tmem_st_32x32b_x32(ts + c0, o);
            }
            ptx::tmem_st_wait();
            load_row();
          }
        }
        ptx::tc_fence_before();
        tc_arrive(bar_sfree + 8 * t, lane);
        if constexpr (SCORED) {
          if (poly) {
            // no key of the tile behind a row, or all: the bias is linear, in groups of
            // eight keys the same up to a step that the maximum and the exponent add
            const bool behind = __all_sync(0xffffffffu, pos <= j0);
            if (behind ||
                __all_sync(0xffffffffu, a.slopes == nullptr || pos - j0 >= TC_KV - 1)) {
              const float sl = behind ? -slope : slope, base = -sl * (float)(pos - j0);
              TcF2 b[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                b[e] = tc_pk(fmaf(sl, (float)(2 * e), base), fmaf(sl, (float)(2 * e + 1), base));
              step = 8.f * sl;
              if (__all_sync(0xffffffffu, big <= poly2_max)) {
#pragma unroll
                for (int c = 0; c < 128; c += 2) {
                  const TcF2 x = tc_pk(s[c], s[c + 1]), v = tc_mul2(x, x);
                  const TcF2 q = tc_fma2(v, tc_fma2(v, low2, low1), low0);
                  tc_un(tc_fma2(x, q, b[(c >> 1) & 3]), s[c], s[c + 1]);
                }
              } else {
#pragma unroll
                for (int c = 0; c < 128; c += 2)
                  tc_un(capped_add(s[c], s[c + 1], b[(c >> 1) & 3]), s[c], s[c + 1]);
              }
            } else {
              const TcF2 d2 = tc_pk1((float)(pos - j0));
#pragma unroll
              for (int c = 0; c < 128; c += 2) {
                float t0, t1;
                tc_un(tc_add2(d2, tc_pk((float)-c, (float)(-c - 1))), t0, t1);
                tc_un(capped(s[c], s[c + 1]), s[c], s[c + 1]);
                s[c] = fmaf(-slope, fabsf(t0), s[c]);
                s[c + 1] = fmaf(-slope, fabsf(t1), s[c + 1]);
              }
            }
          }
        }
        if (!full) {
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c >= lim) s[c] = -INFINITY;
        }
        float mx;
        if constexpr (SCORED) {
          float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
          for (int c = 0; c < 128; c += 8) {
            float y = tc_max3(s[c], s[c + 1], s[c + 2]);
            y = tc_max3(y, s[c + 3], s[c + 4]);
            const float w = tc_max3(s[c + 5], s[c + 6], s[c + 7]);
            y = fmaxf(y, w) + step * (float)(c / 8);
            if (c & 8) x0 = fmaxf(x0, y); else x1 = fmaxf(x1, y);
          }
          mx = fmaxf(x0, x1);
        } else {
          float x0 = s[0], x1 = s[1], x2 = s[2], x3 = s[3];
#pragma unroll
          for (int c = 4; c < 124; c += 8) {
            x0 = tc_max3(x0, s[c], s[c + 1]);
            x1 = tc_max3(x1, s[c + 2], s[c + 3]);
            x2 = tc_max3(x2, s[c + 4], s[c + 5]);
            x3 = tc_max3(x3, s[c + 6], s[c + 7]);
          }
          x0 = tc_max3(x0, s[124], s[125]);
          x1 = tc_max3(x1, s[126], s[127]);
          mx = fmaxf(fmaxf(x0, x1), fmaxf(x2, x3)) * mul;
        }
        if (__any_sync(0xffffffffu, mx > m + TC_LAZY)) {
          float alpha = 1.f;
          if (mx > m + TC_LAZY) {  // also the first keys of the row (m = -inf)
            if (m != -INFINITY) alpha = tc_exp2(m - mx);
            m = mx;
            l *= alpha;
          }
          if (k > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
            tc_wait(bar_pv + 8 * t, (uint32_t)(k - 1) & 1u, tmo, abort_flag);
            ptx::tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              ptx::tmem_ld_32x32b_x16(to + c, o);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; e += 4)
                asm volatile("" : "+r"(o[e]), "+r"(o[e + 1]), "+r"(o[e + 2]), "+r"(o[e + 3]));
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              ptx::tmem_st_32x32b_x16(to + c, o);
            }
          }
        }
        const float mu = m == -INFINITY ? 0.f : m;
        const TcF2 mul2 = tc_pk(mul, mul), mu2 = tc_pk(-mu, -mu);
        TcF2 la = tc_pk(0.f, 0.f), lb = la;
        // P of 64 keys at a time, so that PV starts while the rest is made
        auto weights = [&](int hf, auto poly) {
#pragma unroll
          for (int c = 64 * hf; c < 64 * hf + 64; c += 2) {
            float y0, y1;
            if constexpr (SCORED)
              tc_un(tc_add2(tc_pk(s[c], s[c + 1]), tc_pk1(fmaf(step, (float)(c / 8), -mu))),
                    y0, y1);
            else
              tc_un(tc_fma2(tc_pk(s[c], s[c + 1]), mul2, mu2), y0, y1);
            // one pair of four on the FMA pipe: the special-function pipe, 16
            // results a cycle and SM, is the narrower one (four prompts of 4096
            // tokens, 128-wide heads: none 597 us, 1/8 570, 1/4 561, 3/8 563;
            // where keys are masked all on the latter, for weights of exactly 0; capped
            // or biased scores use the FMA pipe enough, 12 us less for the documents
            // above)
            if (decltype(poly)::value && (c & 6) == 4) {
              tc_un(tc_poly_exp2(y0, y1), y0, y1);
            } else {
              y0 = tc_exp2(y0);
              y1 = tc_exp2(y1);
            }
            if (c & 2) la = tc_add2(la, tc_pk(y0, y1)); else lb = tc_add2(lb, tc_pk(y0, y1));
            u[c >> 1] = Ty::pack(y0, y1);
          }
        };
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          if (full && !SCORED) weights(hf, std::true_type()); else weights(hf, std::false_type());
          if (hf == 0 && k > 0) {  // P of the tile before has been read
            tc_wait(bar_pv + 8 * t, (uint32_t)(k - 1) & 1u, tmo, abort_flag);
            ptx::tc_fence_after();
          }
          ptx::tmem_st_32x32b_x32(tp + 32 * hf, u + 32 * hf);
          ptx::tmem_st_wait();
          ptx::tc_fence_before();
          tc_arrive((hf ? bar_p2 : bar_p) + 8 * t, lane);
        }
        {
          float l0, l1;
          tc_un(tc_add2(la, lb), l0, l1);
          l += l0 + l1;
        }
      }
      tc_wait(bar_pv + 8 * t, (uint32_t)(cnt - 1) & 1u, tmo, abort_flag);
      ptx::tc_fence_after();
    }
    // ---- O / l, or the split's part of it, through the shared memory of the warp's
    // rows of Q (all scores are made): 8 lanes store 128 bytes of a row together.
    // Every lane takes part in the TMEM loads; a half without rows, and a row behind
    // the last, stores nothing.
    if (half_on) {
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no key: 0; NaN stays
      const int64_t prow = (int64_t)z * parts.rows + (int64_t)tok * a.Hq + h;
      const bool part = parts.o != nullptr;
      if (part && real) parts.lse[prow] = l == 0.f ? -INFINITY : m + log2f(l);
      // offset of this thread's row; -1: nothing to store
      const int64_t off = !real ? -1 : part ? (l == 0.f ? -1 : prow * D)
                                            : tok * a.o_ts + (int64_t)h * a.o_hs;
      int64_t ro[8];  // of the rows that this lane stores a piece of
#pragma unroll
      for (int e = 0; e < 8; ++e) ro[e] = __shfl_sync(0xffffffffu, off, 4 * e + (lane >> 3));
      const uint32_t wr = ptx::smem_u32(rows) + lane * 128, rd = ptx::smem_u32(rows);
#pragma unroll 1
      for (int c = 0; c < D; c += 64) {  // 64 columns of E: 128 bytes a row; of fp32: twice
        uint32_t o[64];
        ptx::tmem_ld_32x32b_x32(to + c, o);
        ptx::tmem_ld_32x32b_x32(to + c + 32, o + 32);
        ptx::tmem_ld_wait();
        tc_regs(o);
        tc_regs(o + 32);
        float* f = reinterpret_cast<float*>(o);
#pragma unroll
        for (int e = 0; e < 64; ++e) f[e] = l == 0.f ? 0.f : f[e] * inv;
        if (!part) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            tc_sts(wr + ((e ^ (lane & 7)) << 4), Ty::pack(f[8 * e], f[8 * e + 1]),
                   Ty::pack(f[8 * e + 2], f[8 * e + 3]), Ty::pack(f[8 * e + 4], f[8 * e + 5]),
                   Ty::pack(f[8 * e + 6], f[8 * e + 7]));
          __syncwarp();
          E* const dst = reinterpret_cast<E*>(a.out) + c + 8 * (lane & 7);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int row = 4 * e + (lane >> 3);
            const uint4 v = tc_lds(rd + row * 128 + (((lane & 7) ^ (row & 7)) << 4));
            if (ro[e] >= 0) *reinterpret_cast<uint4*>(dst + ro[e]) = v;
          }
          __syncwarp();
        } else {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              tc_sts(wr + ((e ^ (lane & 7)) << 4), o[32 * q + 4 * e], o[32 * q + 4 * e + 1],
                     o[32 * q + 4 * e + 2], o[32 * q + 4 * e + 3]);
            __syncwarp();
            float* const dst = parts.o + c + 32 * q + 4 * (lane & 7);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int row = 4 * e + (lane >> 3);
              const uint4 v = tc_lds(rd + row * 128 + (((lane & 7) ^ (row & 7)) << 4));
              if (ro[e] >= 0) *reinterpret_cast<uint4*>(dst + ro[e]) = v;
            }
            __syncwarp();
          }
        }
      }
    }
  } else {
    ptx::reg_dec<TC_REG_ISSUE>();
    if (warp == 8) {
    // -------------------------------------------------------------------- TMA
    static_assert(TC_KV == 1 << 7, "boxes of a tile by shifts");
    const int bs = min(a.c.page_shift, 7), br = 1 << bs;           // rows of a box
    const int box = lane & ((TC_KV >> bs) - 1), dh = lane >> (7 - bs);  // this lane's
    const int* own = a.table + (int64_t)r * a.table_stride;
    int g_ring = 0;
    // page number and row of this lane's box of tile k (looked up a tile ahead:
    // the table read takes as long as a tile's softmax)
    auto look = [&](int k, int& page, int& prow) {
      const bool shared = lo + k < np;
      const int off = (shared ? (lo + k) : (lo + k - np)) * TC_KV + box * br;  // in its list
      prow = off & ((1 << a.c.page_shift) - 1);
      page = -1;
      if (k >= cnt || dh >= D / 64 || box * br >= limit(k) - key0(k)) return false;
      page = (shared ? a.prefix_pages : own)[off >> a.c.page_shift];
      return true;
    };
    int page, prow;
    bool mine = look(0, page, prow);
    for (int k = 0; k < cnt; ++k) {
      int page1, prow1;
      const bool mine1 = look(k + 1, page1, prow1);
      if (mine) mine = pg_check(a.c, page) >= 0;
      const uint32_t bytes = (uint32_t)__popc(__ballot_sync(0xffffffffu, mine)) * br * 128u;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv, ++g_ring) {
        const int s = g_ring % L::ST;
        tc_wait(bar_empty + 8 * s, ((uint32_t)(g_ring / L::ST) & 1u) ^ 1u, tmo, abort_flag);
        if (*abort_flag) break;  // (no copy into a stage that is still in use)
        if (lane == 0) ptx::mbar_arrive_expect_tx(bar_full + 8 * s, bytes);
        __syncwarp();
        if (mine)
          ptx::tma_load_4d(sbase + L::OFF_RING + s * L::TILE + dh * L::HB + box * br * 128,
                           kv ? &tm_v : &tm_k, dh * 64, prow, g, page, bar_full + 8 * s);
      }
      mine = mine1;
      page = page1;
      prow = prow1;
    }
    if (*abort_flag) {  // copies in flight land before the shared memory goes
      for (int q = g_ring > L::ST ? g_ring - L::ST : 0; q < g_ring; ++q) {
        const long long t0 = clock64();
        while (!ptx::mbar_try_wait(bar_full + 8 * (q % L::ST), (uint32_t)(q / L::ST) & 1u))
          if (clock64() - t0 > (long long)(tmo * 2ull)) break;
      }
    }
    } else if (warp - 9 < halves) {
    // -------------------------------------------------------------------- MMA
    // One warp per half: an iteration's waits, descriptors and MMAs are some
    // hundred dependent instructions, which one warp for both halves did not get
    // through in the time of a softmax (2900 cycles a pair of tiles, whatever the
    // softmax took).  Uniform copies: the loop and every operand of its MMAs are
    // the same for the warp, and the compiler can see it (an MMA whose
    // descriptors come from vector registers took 130 cycles to issue).
    constexpr bool BF = sizeof(E) == 2 && !std::is_same<E, __half>::value;
    constexpr uint32_t id_qk = ptx::idesc_16_f32(TC_HALF, TC_KV, BF, false);
    constexpr uint32_t id_pv = ptx::idesc_16_f32(TC_HALF, D, BF, true);
    const int t = __reduce_max_sync(0xffffffffu, warp - 9);
    const int cnt_u = __reduce_max_sync(0xffffffffu, cnt);
    const int halves_u = __reduce_max_sync(0xffffffffu, halves);
    const uint32_t tm = __reduce_max_sync(0xffffffffu, tmem);
    const uint32_t who = ptx::elect_one();
    const uint64_t dq = ptx::smem_desc_sw128(sbase + t * L::TILE);
    const uint64_t dk = ptx::smem_desc_sw128(sbase + L::OFF_RING);
    const uint64_t dv = ptx::smem_desc_sw128_mn(sbase + L::OFF_RING, L::HB);
    const uint32_t tm_s = tm + L::COL_S, tm_p = tm + L::COL_P + t * 64,
                   tm_o = tm + L::COL_O + t * D;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (ptx::mbar_try_wait_now(bar, parity)) return;
      const long long t0 = clock64();
      while (!ptx::mbar_try_wait_now(bar, parity)) {
        if (*abort_flag || clock64() - t0 > (long long)(tmo * 2ull)) {
          *abort_flag = 1;
          break;
        }
      }
    };
    // the stage is free when both halves are done with it: the only half says so
    // twice
    auto release = [&](int s) {
      ptx::mma_commit_if(who, bar_empty + 8 * s);
      if (halves_u == 1) ptx::mma_commit_if(who, bar_empty + 8 * s);
    };
    // zeros in the rows of stage s behind the first `have`, which may hold anything (or
    // were not loaded); both halves' warps write them, each before its own MMAs
    auto clear = [&](int s, int have) {
      if (have >= TC_KV) return;
      uint8_t* rows = smem + L::OFF_RING + s * L::TILE;
      for (int x = have * 8 + lane; x < TC_KV * 8; x += 32)
#pragma unroll
        for (int hb = 0; hb < D / 64; ++hb)
          *reinterpret_cast<uint4*>(rows + hb * L::HB + x * 16) = make_uint4(0u, 0u, 0u, 0u);
      ptx::fence_proxy_async_smem();
      __syncwarp();
    };
    // K of tile k in stage s.  Scores behind the last key are masked, but how capped ones
    // are computed goes by the largest of a warp's (above): what lies behind a request
    // must not change the bits of its rows.
    auto qk = [&](int k, int s) {
      if (SCORED) clear(s, limit(k) - key0(k));
      const uint64_t b0 = dk + (uint64_t)(s * (L::TILE >> 4));
#pragma unroll
      for (int e = 0; e < D / 16; ++e)
        ptx::mma_f16_ss_if(who, tm_s, dq + ((e >> 2) * L::HB + (e & 3) * 32) / 16,
                           b0 + ((e >> 2) * L::HB + (e & 3) * 32) / 16, id_qk, e != 0 ? 1u : 0u);
      if (!skip_signal) ptx::mma_commit_if(who, bar_s + 8 * t);
      release(s);
    };
    wait(bar_q, 0);
    wait(bar_full, 0);
    // half 1's first scores go where half 0's were, once those have been read
    if (t == 1) {
      wait(bar_sfree, 0);
      ptx::tc_fence_after();
    }
    qk(0, 0);
    int sk = 2 % L::ST, sv = 1;       // stages of K of the next tile and V of this one
    uint32_t phk = 0, phv = 0, par = 0;
#pragma unroll 1
    for (int k = 0; k < cnt_u; ++k, par ^= 1u) {
      wait(bar_full + 8 * sv, phv);
      // V's rows behind the last key: their weights are zero, and 0 x NaN is NaN
      clear(sv, limit(k) - key0(k));
      if (k + 1 < cnt_u) {
        wait(bar_full + 8 * sk, phk);
        // S is free once the other half has read it (half 1 of this tile; half 0 of
        // the next), or this one where there is no other
        if (halves_u == 2)
          wait(bar_sfree + 8 * (1 - t), t == 0 ? par : par ^ 1u);
        else
          wait(bar_sfree, par);
        ptx::tc_fence_after();
        qk(k + 1, sk);
      }
      const uint64_t b0 = dv + (uint64_t)(sv * (L::TILE >> 4));
      wait(bar_p + 8 * t, par);
      ptx::tc_fence_after();
#pragma unroll
      for (int e = 0; e < 4; ++e)
        ptx::mma_f16_ts_if(who, tm_o, tm_p + e * 8, b0 + e * 128, id_pv, (k | e) != 0 ? 1u : 0u);
      wait(bar_p2 + 8 * t, par);
      ptx::tc_fence_after();
#pragma unroll
      for (int e = 4; e < 8; ++e)
        ptx::mma_f16_ts_if(who, tm_o, tm_p + e * 8, b0 + e * 128, id_pv, 1u);
      ptx::mma_commit_if(who, bar_pv + 8 * t);
      release(sv);
      sk += 2;
      if (sk >= L::ST) {
        sk -= L::ST;
        phk ^= 1u;
      }
      sv += 2;
      if (sv >= L::ST) {
        sv -= L::ST;
        phv ^= 1u;
      }
    }
    __syncwarp();
    if (*abort_flag) {  // MMAs in flight end before their memory goes
      ptx::mma_commit_if(who, bar_drain + 8 * t);
      const long long t0 = clock64();
      while (!ptx::mbar_try_wait(bar_drain + 8 * t, 0))
        if (clock64() - t0 > (long long)(tmo * 2ull)) break;
    }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) pg_error(a.c, DDQ_ERR_TIMEOUT);
  if (warp == 9) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
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
  if (row >= p.rows) return;  // rows < 2^31
  const int t = (int)((uint32_t)row / (uint32_t)a.Hq), h = (int)row - t * a.Hq;
  if (a.cu && (t < a.cu[0] || t >= a.cu[a.R])) return;  // a padded row stays as it is
  // four parts in flight together, the first ones while the maximum is found (a part
  // without keys was not written: its values are dropped)
  float v[4][DPL], ls[4];
  auto load = [&](int z0) {
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int z = min(z0 + y, p.count - 1);
      const float* src = p.o + (z * p.rows + row) * D + lane * DPL;
      if constexpr (DPL == 2)
        *reinterpret_cast<float2*>(v[y]) = *reinterpret_cast<const float2*>(src);
      else
        *reinterpret_cast<float4*>(v[y]) = *reinterpret_cast<const float4*>(src);
      ls[y] = z0 + y < p.count ? p.lse[z * p.rows + row] : -INFINITY;
    }
  };
  load(0);
  float mx = -INFINITY;
  for (int z = lane; z < p.count; z += 32) mx = fmaxf(mx, p.lse[z * p.rows + row]);
  mx = warp_max(mx);
  float den = 0.f, o[DPL];
#pragma unroll
  for (int e = 0; e < DPL; ++e) o[e] = 0.f;
  for (int z = 0; z < p.count;) {
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const float w = ls[y] == -INFINITY ? 0.f : exp2f(ls[y] - mx);
      den += w;
#pragma unroll
      for (int e = 0; e < DPL; ++e) o[e] = fmaf(w, w != 0.f ? v[y][e] : 0.f, o[e]);
    }
    z += 4;
    if (z < p.count) load(z);
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

namespace {
PFN_cuTensorMapEncodeTiled_v12000 tc_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}
}  // namespace

// The pool as {D, page, Hkv, pages} with boxes of 64 dimensions x `rows` rows.
int pg_tensor_map(CUtensorMap* m, const PgCache& c, const void* base, bool bf16, int rows) {
  auto enc = tc_encoder();
  if (!enc) return DDQ_ERR_DEVICE;
  cuuint64_t dims[4] = {(cuuint64_t)c.D, (cuuint64_t)1 << c.page_shift, (cuuint64_t)c.Hkv,
                        (cuuint64_t)c.num_pages};
  cuuint64_t strides[3] = {(cuuint64_t)c.row_stride * 2, (cuuint64_t)c.head_stride * 2,
                           (cuuint64_t)c.page_stride * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r =
      enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
          const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? DDQ_OK : DDQ_ERR_SHAPE;
}

// The most tiles that T rows of R requests make (a request ends inside a tile).
int64_t tc_tiles(int64_t T, int64_t R, int64_t G, bool ragged) {
  if (!ragged) return (T * G + TC_ROWS - 1) / TC_ROWS;
  return T * G / TC_ROWS + (R < T ? R : T);
}

// Splits of the key axis, where the CTAs would not fill the GPU: the number with the
// least of rounds x (key tiles of a CTA + 3 for its start and end) plus the parts'
// way through memory (a tile takes about 1.5 us, in which 9 MB pass) and, for
// prompts, the joining kernel, which a decode step has anyway.  The keys are those
// that the table's width could hold, for the lengths are on the device: with a table
// much wider than the requests, short ones are split too (8 prompts of 512 tokens,
// 20 us, take 51 with a table for 32768 keys).
int tc_splits(int64_t T, int64_t R, int Hq, int Hkv, int64_t keys, bool ragged, int sms) {
  const int64_t ctas = tc_tiles(T, R, Hq / Hkv, ragged) * Hkv;
  const int64_t nt = (keys + TC_KV - 1) / TC_KV;
  const double part = (double)T * Hq * 128 * 8 / 9e6;
  int best = 1;
  double least = 0;
  for (int s = 1; s <= 64 && s <= nt; ++s) {
    const double rounds = (double)((ctas * s + sms - 1) / sms);
    const double cost = rounds * (double)((nt + s - 1) / s + 3) +
                        (s > 1 || !ragged ? s * part : 0) + (s > 1 && ragged ? 2 : 0);
    if (s == 1 || cost < least) {
      least = cost;
      best = s;
    }
    if (s == 1 && ctas >= 4 * (int64_t)sms) break;
  }
  return best;
}

int launch_paged_tc(const PgAttnArgs& a, bool bf16, const PgParts& parts, int splits,
                    unsigned long long tmo, int debug_flags, cudaStream_t s) {
  const int G = a.G;
  const int64_t tiles = tc_tiles(a.T, a.R, G, a.cu != nullptr);
  if (tiles > 0x7fffffff / a.c.Hkv) return DDQ_ERR_SHAPE;
  CUtensorMap tk, tv;
  const int br = (1 << a.c.page_shift) < TC_KV ? (1 << a.c.page_shift) : TC_KV;
  int st = pg_tensor_map(&tk, a.c, a.c.k, bf16, br);
  if (!st) st = pg_tensor_map(&tv, a.c, a.c.v, bf16, br);
  if (st) return st;
  const int dev = current_device();
  static SmemAttrOnce attr[2][2][2];
  const bool scored = a.cap > 0.f || a.slopes != nullptr || !(a.scale > 0.f);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * a.c.Hkv), (unsigned)splits);
  cfg.blockDim = dim3(TC_NT);
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
    // test hook (ddq_set_debug bit 0): no scores-ready signal, so that the softmax's
    // bounded waits run out and every role winds down
    e = cudaLaunchKernelEx(&cfg, kern, tk, tv, a, parts, splits, debug_flags & 1, tmo);
    return DDQ_OK;
  };
#define DDQ_TC(E_, D_, B_)                                                                      \
  (scored ? go(paged_tc_kernel<E_, D_, true>, attr[D_ / 128][B_][1], TcLayout<D_>::SMEM)        \
          : go(paged_tc_kernel<E_, D_, false>, attr[D_ / 128][B_][0], TcLayout<D_>::SMEM))
  if (a.c.D == 64)
    st = bf16 ? DDQ_TC(__nv_bfloat16, 64, 1) : DDQ_TC(__half, 64, 0);
  else
    st = bf16 ? DDQ_TC(__nv_bfloat16, 128, 1) : DDQ_TC(__half, 128, 0);
#undef DDQ_TC
  if (st) return st;
  if (e != cudaSuccess) {
    cudaGetLastError();
    return DDQ_ERR_LAUNCH;
  }
  return check_launch();
}

}  // namespace ddq
