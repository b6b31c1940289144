// capi.cu - the extern "C" entry points declared in include/ddq_b200.h:
// argument validation, per-device attribute cache and kernel dispatch.
#include <cstdlib>
#include <mutex>

#include "common.cuh"
#include "launch.cuh"

namespace ddq {

namespace {
constexpr int kMaxDevices = 64;
int g_sm_count[kMaxDevices];
std::once_flag g_sm_once[kMaxDevices];
}  // namespace

int current_device() {
  int d = 0;
  if (cudaGetDevice(&d) != cudaSuccess) return -1;
  return d;
}

int device_sm_count(int device) {
  if (device < 0 || device >= kMaxDevices) return -1;
  std::call_once(g_sm_once[device], [device] {
    int v = 0;
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) v = -1;
    g_sm_count[device] = v;
  });
  return g_sm_count[device];
}

// Programmatic dependent launch for the tensor-core kernels (on unless
// DDQ_NO_PDL is set, which exists to measure what it buys).
bool pdl_enabled() {
  static bool v = std::getenv("DDQ_NO_PDL") == nullptr;
  return v;
}

int check_launch() {
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? DDQ_OK : DDQ_ERR_LAUNCH;
}

int* device_error_word() {
  static std::once_flag once[kMaxDev];
  static int* ptr[kMaxDev];
  const int d = current_device();
  if (d < 0 || d >= kMaxDev) return nullptr;
  std::call_once(once[d], [d] {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_device_error) != cudaSuccess) {
      cudaGetLastError();
      p = nullptr;
    }
    ptr[d] = static_cast<int*>(p);
  });
  return ptr[d];
}

namespace {
// Kernel choice by M: M < tc_min_m -> CUDA-core skinny kernel; M <= 64 ->
// decode kernel (e4m3 tensor cores, activation planes); M > 64 -> prefill
// kernel (fp16 tensor cores on converted weight tiles).  DDQ_TC_MIN_M
// overrides the first threshold for benchmarking.
int tc_min_m() {
  static int v = [] {
    const char* e = std::getenv("DDQ_TC_MIN_M");
    int x = e ? std::atoi(e) : 1;
    return x < 1 ? 1 : x;
  }();
  return v;
}
constexpr int64_t kDecodeMaxM = 64;

// Up to this many tokens a GEMM whose shape thin.cu takes runs the
// shared-memory-resident mma.sync kernel instead of the e4m3 decode kernel.
// DDQ_THIN_MAX_M overrides (0 switches it off) for benchmarking.
int64_t thin_max_m() {
  static const int64_t v = [] {
    const char* e = std::getenv("DDQ_THIN_MAX_M");
    return e ? (int64_t)std::atoll(e) : (int64_t)16;
  }();
  return v;
}

// From this many tokens on, a GEMM expands the weights to fp16 once and runs
// the fp16 tensor-core GEMM (tc_prefill.cu); between kDecodeMaxM and this the
// in-kernel conversion of tc_gemm.cu is cheaper.  DDQ_PF_MIN_M overrides.
int64_t pf_min_m() {
  static const int64_t v = [] {
    const char* e = std::getenv("DDQ_PF_MIN_M");
    return e ? (int64_t)std::atoll(e) : (int64_t)128;
  }();
  return v;
}
bool pf_shape(int64_t M, int64_t N) { return M > kDecodeMaxM && M >= pf_min_m() && N % 8 == 0; }

// Test hooks (ddq_set_debug): bounded-wait limit and fault-injection flags.
unsigned long long g_wait_timeout_ns = 1000000000ull;  // 1 s
int g_debug_flags = 0;

// The thin kernel has no fault-injection hook, so while a test sets the
// injection flag (bit 0) or asks for the split + decode kernels (bit 2), the
// shapes it would take run the decode kernel; the trace flag (bit 1), the
// thin-kernel test flag (bit 3) and the tensor-core resident-slice flag
// (bit 6, which takes no 1..16-token shape) keep it (it writes phase stamps
// too).
bool thin_shape(int64_t M, int64_t N, int64_t K) {
  if (M > thin_max_m() || (g_debug_flags & ~(2 | 8 | 64 | 128)) != 0) return false;
  const int dev = current_device();
  return dev >= 0 && thin_eligible(M, N, K, device_sm_count(dev));
}

// The resident-slice kernel (rs.cu) takes the shapes it fits first, under
// the same debug-flag rule as the thin kernel; bit 3 sends its shapes to the
// thin kernel (which then takes the ones it fits); bit 6 (the tensor-core
// resident-slice kernel for 17..64 tokens) leaves both of them in place.
bool rs_shape(int64_t M, int64_t N, int64_t K) {
  if ((g_debug_flags & ~(2 | 64 | 128)) != 0) return false;
  const int dev = current_device();
  return dev >= 0 && rs_eligible(M, N, K, device_sm_count(dev));
}

// The tensor-core resident-slice kernel (rt.cu) is opt-in (debug bit 6): in
// a chain of dependent calls it measured slower than the mma.sync resident
// slice and the split + e4m3 decode kernels at every Qwen2.5 shape (e.g.
// q/k/v at 64 tokens 7.3 vs 4.9 us, gate/up 11.9 vs 7.8 us).  With the bit
// it takes 17..64-token shapes before every other path; any further bit but
// the trace (1) and its timeout hook (4) sends them to the older paths.
bool rt_shape(int64_t M, int64_t N, int64_t K, bool swiglu) {
  if ((g_debug_flags & 64) == 0 || (g_debug_flags & ~(2 | 16 | 64 | 128)) != 0) return false;
  const int dev = current_device();
  return dev >= 0 && rt_eligible(M, N, K, device_sm_count(dev), swiglu);
}

bool tc_eligible(const void* x, const void* wq, int64_t K) {
  return K > 0 && (K % 16 == 0) && aligned16(x) && aligned16(wq);
}
}  // namespace

unsigned long long wait_timeout_ns() { return g_wait_timeout_ns; }
int debug_flags() { return g_debug_flags; }

}  // namespace ddq

using namespace ddq;

extern "C" const char* ddq_status_string(int status) {
  switch (status) {
    case DDQ_OK: return "ok";
    case DDQ_ERR_INVALID_ARGUMENT: return "invalid argument (null pointer or bad dtype code)";
    case DDQ_ERR_SHAPE: return "unsupported or inconsistent shape";
    case DDQ_ERR_ALIGNMENT: return "pointer alignment not supported";
    case DDQ_ERR_WORKSPACE: return "workspace missing or too small";
    case DDQ_ERR_DEVICE: return "no usable sm_100 device";
    case DDQ_ERR_LAUNCH: return "CUDA kernel launch failed";
    case DDQ_ERR_TIMEOUT: return "device-side bounded wait timed out";
    case DDQ_ERR_PAGE: return "page, slot, length or position outside the paged cache";
    default: return "unknown ddq status";
  }
}

extern "C" int ddq_version(void) { return (0 << 16) | 1; }

extern "C" size_t ddq_w8a16_gemm_workspace_size(int64_t M, int64_t N, int64_t K) {
  if (M < tc_min_m() || M <= 0 || N <= 0 || K <= 0 || K % 16 != 0) return 0;
  const int dev = current_device();
  const int sms = dev >= 0 ? device_sm_count(dev) : -1;
  if (M <= kDecodeMaxM) return dec_plan(M, N, K, sms > 0 ? sms : 148).ws_bytes;
  if (pf_shape(M, N)) return 2 * pf_workspace_bytes(N, K);  // two alternating buffers
  return tc_plan(M, N, K, sms > 0 ? sms : 148).ws_bytes;
}

extern "C" int ddq_w8a16_gemm(const void* x, const uint8_t* wq, const float* scales,
                              const void* bias, int bias_dtype, void* y, int64_t M, int64_t N,
                              int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  (void)workspace; (void)workspace_bytes;
  if (M < 0 || N < 0 || K < 0) return DDQ_ERR_SHAPE;
  if (bias_dtype != DDQ_DTYPE_NONE && bias_dtype != DDQ_DTYPE_F16 && bias_dtype != DDQ_DTYPE_F32)
    return DDQ_ERR_INVALID_ARGUMENT;
  if (bias_dtype != DDQ_DTYPE_NONE && !bias) return DDQ_ERR_INVALID_ARGUMENT;
  if (M == 0 || N == 0) return DDQ_OK;
  if (!x || !wq || !scales || !y) return DDQ_ERR_INVALID_ARGUMENT;
  if (M > 0x7fffffff || N > 0x7fffffff || K > 0x7fffffff) return DDQ_ERR_SHAPE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const __half* xh = reinterpret_cast<const __half*>(x);
  __half* yh = reinterpret_cast<__half*>(y);
  if (tc_eligible(x, wq, K) && M >= tc_min_m()) {
    if (rt_shape(M, N, K, false))
      return launch_rt(xh, wq, scales, bias, bias_dtype, yh, (int)M, (int)N, (int)K, false,
                       g_wait_timeout_ns, s, g_debug_flags);
    if (rs_shape(M, N, K))
      return launch_rs(xh, wq, scales, bias, bias_dtype, yh, (int)M, (int)N, (int)K,
                       g_wait_timeout_ns, s, g_debug_flags);
    if (thin_shape(M, N, K))
      return launch_thin(xh, wq, scales, bias, bias_dtype, yh, (int)M, (int)N, (int)K,
                         g_wait_timeout_ns, s, g_debug_flags);
    if (M <= kDecodeMaxM)
      return launch_dec(xh, wq, scales, bias, bias_dtype, yh, nullptr, 0, (int)M, (int)N, (int)K,
                        workspace, workspace_bytes, g_wait_timeout_ns, g_debug_flags, s);
    if (pf_shape(M, N) && aligned16(y) && workspace &&
        workspace_bytes >= pf_workspace_bytes(N, K))
      return launch_pf(xh, wq, scales, bias, bias_dtype, yh, (int)M, (int)N, (int)K, workspace,
                       workspace_bytes, g_wait_timeout_ns, g_debug_flags, s);
    return launch_tc(xh, wq, scales, bias, bias_dtype, yh, nullptr, 0, (int)M, (int)N, (int)K,
                     workspace, workspace_bytes, g_wait_timeout_ns, g_debug_flags, s);
  }
  const bool fast = tc_eligible(x, wq, K) && K <= 12288;
  if (!fast) return launch_generic(xh, wq, scales, bias, bias_dtype, yh, M, N, K, s);
  return launch_skinny(xh, wq, scales, bias, bias_dtype, yh, (int)M, (int)N, (int)K, s);
}

extern "C" int ddq_w8a16_gemm_kernel_count(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  if (K % 16 != 0 || M < tc_min_m()) return 1;
  if (rt_shape(M, N, K, false) || rs_shape(M, N, K) || thin_shape(M, N, K)) return 1;
  if (M <= kDecodeMaxM || pf_shape(M, N)) return 2;  // split + GEMM / expansion + GEMM
  return 1;
}

extern "C" size_t ddq_w8a16_gemm_swiglu_workspace_size(int64_t M, int64_t I, int64_t K) {
  if (M <= 0 || I <= 0 || K <= 0 || K % 16 != 0 || I % 16 != 0) return 0;
  const int dev = current_device();
  const int sms = dev >= 0 ? device_sm_count(dev) : -1;
  if (M <= kDecodeMaxM) return dec_plan(M, 2 * I, K, sms > 0 ? sms : 148, true).ws_bytes;
  return 2 * pf_workspace_bytes(2 * I, K);  // two alternating buffers
}

extern "C" int ddq_w8a16_gemm_swiglu(const void* x, const uint8_t* wq_gu, const float* scales_gu,
                                     const void* bias, int bias_dtype, void* z, int64_t M,
                                     int64_t I, int64_t K, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  if (M < 0 || I < 0 || K < 0) return DDQ_ERR_SHAPE;
  if (bias_dtype != DDQ_DTYPE_NONE && bias_dtype != DDQ_DTYPE_F16 && bias_dtype != DDQ_DTYPE_F32)
    return DDQ_ERR_INVALID_ARGUMENT;
  if (bias_dtype != DDQ_DTYPE_NONE && !bias) return DDQ_ERR_INVALID_ARGUMENT;
  if (M == 0 || I == 0) return DDQ_OK;
  if (!x || !wq_gu || !scales_gu || !z) return DDQ_ERR_INVALID_ARGUMENT;
  if (I % 16 != 0 || K == 0 || K % 16 != 0 || M > 0x7fffffff || 2 * I > 0x7fffffff ||
      K > 0x7fffffff)
    return DDQ_ERR_SHAPE;
  if (!aligned16(x) || !aligned16(wq_gu) || !aligned16(z)) return DDQ_ERR_ALIGNMENT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const __half* xh = reinterpret_cast<const __half*>(x);
  __half* zh = reinterpret_cast<__half*>(z);
  if (M >= tc_min_m() && rt_shape(M, 2 * I, K, true))
    return launch_rt(xh, wq_gu, scales_gu, bias, bias_dtype, zh, (int)M, (int)(2 * I), (int)K,
                     true, g_wait_timeout_ns, s, g_debug_flags);
  if (M <= kDecodeMaxM)
    return launch_dec(xh, wq_gu, scales_gu, bias, bias_dtype, zh, nullptr, 0, (int)M, (int)(2 * I),
                      (int)K, workspace, workspace_bytes, g_wait_timeout_ns, g_debug_flags, s,
                      true);
  return launch_pf(xh, wq_gu, scales_gu, bias, bias_dtype, zh, (int)M, (int)(2 * I), (int)K,
                   workspace, workspace_bytes, g_wait_timeout_ns, g_debug_flags, s, true);
}

extern "C" int ddq_prefill_rope_kv(const void* qkv, int64_t qkv_stride, void* k_cache,
                                   void* v_cache, int64_t cache_batch_stride, int64_t capacity,
                                   const float* cos, const float* sin, int64_t start,
                                   void* q_out, void* k_out, void* v_out, int64_t B, int64_t S,
                                   int64_t Hq, int64_t Hkv, int64_t D, void* stream) {
  if (B < 0 || S < 0 || Hq < 0 || Hkv < 0 || capacity < 0 || start < 0) return DDQ_ERR_SHAPE;
  if (B == 0 || S == 0) return DDQ_OK;
  if (!qkv || !k_cache || !v_cache || !cos || !sin || !q_out) return DDQ_ERR_INVALID_ARGUMENT;
  if (Hq < 1 || Hkv < 1 || B * S > 0x7fffffffll || Hq > 1024 || Hkv > 1024 ||
      capacity > 0x7fffffff || start + S > capacity || qkv_stride < (Hq + 2 * Hkv) * D ||
      cache_batch_stride < Hkv * capacity * D)
    return DDQ_ERR_SHAPE;
  return launch_prefill_rope_kv(
      reinterpret_cast<const __half*>(qkv), qkv_stride, reinterpret_cast<__half*>(k_cache),
      reinterpret_cast<__half*>(v_cache), cache_batch_stride, (int)capacity, cos, sin,
      (int)start, reinterpret_cast<__half*>(q_out), reinterpret_cast<__half*>(k_out),
      reinterpret_cast<__half*>(v_out), (int)B, (int)S, (int)Hq, (int)Hkv, (int)D,
      reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int ddq_w8a16_gemm_qkv_rope_kv(const void* x, const uint8_t* wq, const float* scales,
                                          const void* bias, int bias_dtype, int64_t B, int64_t S,
                                          int64_t K, int64_t Hq, int64_t Hkv, int64_t D,
                                          void* k_cache, void* v_cache,
                                          int64_t cache_batch_stride, int64_t capacity,
                                          const float* cos, const float* sin, int64_t start,
                                          void* q_out, void* k_out, void* v_out, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  if (B < 0 || S < 0 || K < 0 || Hq < 0 || Hkv < 0 || capacity < 0 || start < 0)
    return DDQ_ERR_SHAPE;
  if (bias_dtype != DDQ_DTYPE_NONE && bias_dtype != DDQ_DTYPE_F16 && bias_dtype != DDQ_DTYPE_F32)
    return DDQ_ERR_INVALID_ARGUMENT;
  if (bias_dtype != DDQ_DTYPE_NONE && !bias) return DDQ_ERR_INVALID_ARGUMENT;
  if (B == 0 || S == 0) return DDQ_OK;
  if (!x || !wq || !scales || !k_cache || !v_cache || !cos || !sin || !q_out)
    return DDQ_ERR_INVALID_ARGUMENT;
  const int64_t M = B * S, N = (Hq + 2 * Hkv) * D;
  // the fused epilogue's shapes only (head_dim 64, a prefill-size chunk);
  // callers run the GEMM and ddq_prefill_rope_kv for the others
  if (D != 64 || Hq < 1 || Hkv < 1 || K == 0 || K % 16 != 0 || M > 0x7fffffff ||
      N > 0x7fffffff || K > 0x7fffffff || capacity > 0x7fffffff || !pf_shape(M, N))
    return DDQ_ERR_SHAPE;
  if (start + S > capacity || cache_batch_stride < Hkv * capacity * D) return DDQ_ERR_SHAPE;
  // the epilogue reads cos/sin and writes q, k, v by whole 32-byte sectors
  auto a32 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; };
  if (!aligned16(x) || !aligned16(wq) || !a32(q_out) || !a32(k_cache) || !a32(v_cache) ||
      (k_out && !a32(k_out)) || (v_out && !a32(v_out)) || !a32(cos) || !a32(sin) ||
      cache_batch_stride % 16 != 0)
    return DDQ_ERR_ALIGNMENT;
  PfRope r{};
  r.kc = reinterpret_cast<__half*>(k_cache);
  r.vc = reinterpret_cast<__half*>(v_cache);
  r.cache_bstride = cache_batch_stride;
  r.cap = (int)capacity;
  r.cos = cos;
  r.sin = sin;
  r.start = (int)start;
  r.q_out = reinterpret_cast<__half*>(q_out);
  r.k_out = reinterpret_cast<__half*>(k_out);
  r.v_out = reinterpret_cast<__half*>(v_out);
  r.S = (int)S;
  r.Hq = (int)Hq;
  r.Hkv = (int)Hkv;
  return launch_pf(reinterpret_cast<const __half*>(x), wq, scales, bias, bias_dtype, nullptr,
                   (int)M, (int)N, (int)K, workspace, workspace_bytes, g_wait_timeout_ns,
                   g_debug_flags, reinterpret_cast<cudaStream_t>(stream), false, &r);
}

extern "C" int ddq_decode_attention(const void* qkv, int64_t qkv_stride, void* k_cache,
                                    void* v_cache, int64_t cache_batch_stride, int64_t capacity,
                                    const float* cos, const float* sin, const int64_t* pos,
                                    void* out, int64_t out_stride, int64_t B, int64_t Hq,
                                    int64_t Hkv, int64_t D, float scale, void* stream) {
  if (B < 0 || Hq < 0 || Hkv < 0 || D < 0 || capacity < 0) return DDQ_ERR_SHAPE;
  if (B == 0) return DDQ_OK;
  if (!qkv || !k_cache || !v_cache || !cos || !sin || !pos || !out) return DDQ_ERR_INVALID_ARGUMENT;
  if (B > 65535 || Hq > 1024 || capacity > 0x7fffffff ||
      qkv_stride < (Hq + 2 * Hkv) * D || out_stride < Hq * D ||
      cache_batch_stride < Hkv * capacity * D)
    return DDQ_ERR_SHAPE;
  return launch_decode_attention(
      reinterpret_cast<const __half*>(qkv), qkv_stride, reinterpret_cast<__half*>(k_cache),
      reinterpret_cast<__half*>(v_cache), cache_batch_stride, (int)capacity, cos, sin, pos,
      reinterpret_cast<__half*>(out), out_stride, nullptr, nullptr, (int)B, (int)Hq, (int)Hkv,
      (int)D, scale, g_wait_timeout_ns, g_debug_flags, 0, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int ddq_decode_attention_split(const void* qkv, int64_t qkv_stride, void* k_cache,
                                          void* v_cache, int64_t cache_batch_stride,
                                          int64_t capacity, const float* cos, const float* sin,
                                          const int64_t* pos, void* out, int64_t out_stride,
                                          uint8_t* planes, float* xscale, int64_t B, int64_t Hq,
                                          int64_t Hkv, int64_t D, float scale, int flags,
                                          void* stream) {
  if (B < 0 || Hq < 0 || Hkv < 0 || D < 0 || capacity < 0) return DDQ_ERR_SHAPE;
  if (B == 0) return DDQ_OK;
  if (!qkv || !k_cache || !v_cache || !cos || !sin || !pos || !planes || !xscale)
    return DDQ_ERR_INVALID_ARGUMENT;
  if (B > 65535 || Hq > 1024 || capacity > 0x7fffffff ||
      qkv_stride < (Hq + 2 * Hkv) * D || (out && out_stride < Hq * D) ||
      cache_batch_stride < Hkv * capacity * D)
    return DDQ_ERR_SHAPE;
  return launch_decode_attention(
      reinterpret_cast<const __half*>(qkv), qkv_stride, reinterpret_cast<__half*>(k_cache),
      reinterpret_cast<__half*>(v_cache), cache_batch_stride, (int)capacity, cos, sin, pos,
      reinterpret_cast<__half*>(out), out_stride, planes, xscale, (int)B, (int)Hq, (int)Hkv,
      (int)D, scale, g_wait_timeout_ns, g_debug_flags, flags,
      reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int ddq_add_rmsnorm(const void* x, const void* delta, const float* w, float eps,
                               void* x_out, void* h, int64_t M, int64_t H, void* stream) {
  if (M < 0 || H < 0) return DDQ_ERR_SHAPE;
  if (M == 0) return DDQ_OK;
  if (!x || !w || !h) return DDQ_ERR_INVALID_ARGUMENT;
  if (M > 0x7fffffff || H > 0x7fffffff) return DDQ_ERR_SHAPE;
  return launch_add_rmsnorm(reinterpret_cast<const __half*>(x),
                            reinterpret_cast<const __half*>(delta), w, eps,
                            reinterpret_cast<__half*>(x_out), reinterpret_cast<__half*>(h),
                            (int)M, (int)H, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int ddq_add_rmsnorm_split(const void* x, const void* delta, const float* w, float eps,
                                     void* x_out, void* h, uint8_t* planes, float* xscale,
                                     int64_t M, int64_t H, void* stream) {
  if (M < 0 || H < 0) return DDQ_ERR_SHAPE;
  if (M == 0) return DDQ_OK;
  if (!x || !w || !planes || !xscale) return DDQ_ERR_INVALID_ARGUMENT;
  if (M > 0x7fffffff || H > 0x7fffffff) return DDQ_ERR_SHAPE;
  return launch_add_rmsnorm_split(
      reinterpret_cast<const __half*>(x), reinterpret_cast<const __half*>(delta), w, eps,
      reinterpret_cast<__half*>(x_out), reinterpret_cast<__half*>(h), planes, xscale, (int)M,
      (int)H, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int ddq_w8a16_gemm_planes(const uint8_t* planes, const float* xscale,
                                     const uint8_t* wq, const float* scales, const void* bias,
                                     int bias_dtype, void* y, int64_t M, int64_t N, int64_t K,
                                     int swiglu, void* stream) {
  if (M < 0 || N < 0 || K < 0) return DDQ_ERR_SHAPE;
  if (bias_dtype != DDQ_DTYPE_NONE && bias_dtype != DDQ_DTYPE_F16 && bias_dtype != DDQ_DTYPE_F32)
    return DDQ_ERR_INVALID_ARGUMENT;
  if (bias_dtype != DDQ_DTYPE_NONE && !bias) return DDQ_ERR_INVALID_ARGUMENT;
  if (M == 0 || N == 0) return DDQ_OK;
  if (!planes || !xscale || !wq || !scales || !y) return DDQ_ERR_INVALID_ARGUMENT;
  if (M > kDecodeMaxM || K == 0 || K % 16 != 0 || N > 0x7fffffff || K > 0x7fffffff ||
      (swiglu && N % 32 != 0))
    return DDQ_ERR_SHAPE;
  if (!aligned16(wq) || !aligned16(y)) return DDQ_ERR_ALIGNMENT;
  return launch_dec(nullptr, wq, scales, bias, bias_dtype, reinterpret_cast<__half*>(y), nullptr,
                    0, (int)M, (int)N, (int)K, nullptr, 0, g_wait_timeout_ns, g_debug_flags,
                    reinterpret_cast<cudaStream_t>(stream), swiglu != 0, planes, xscale);
}

extern "C" int ddq_argmax_f16(const void* logits, int64_t B, int64_t V, int64_t* out,
                              void* stream) {
  if (B < 0 || V < 0) return DDQ_ERR_SHAPE;
  if (B == 0) return DDQ_OK;
  if (!logits || !out) return DDQ_ERR_INVALID_ARGUMENT;
  if (V > 0xFFFFFFFFll) return DDQ_ERR_SHAPE;
  return launch_argmax_f16(reinterpret_cast<const __half*>(logits), B, V, out,
                           reinterpret_cast<cudaStream_t>(stream));
}

// The fused lm_head runs token rows in chunks of at most 64 (one tensor-core
// token tile); chunks reuse one workspace in stream order.
static const int64_t kLmChunk = 64;

// Workspace layout of the fused lm_head: [0, lmh_area_bytes) the streaming
// kernel's arrival counter and per-CTA words (kept zero between calls), then
// the decode kernel's activation planes for calls of more tokens.
extern "C" size_t ddq_lm_head_argmax_workspace_size(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || K % 16 != 0) return 0;
  const int64_t mc = M < kLmChunk ? M : kLmChunk;
  const int dev = current_device();
  const int sms = dev >= 0 ? device_sm_count(dev) : -1;
  const size_t area = lmh_area_bytes(sms);
  if (mc < tc_min_m()) return area;
  return area + dec_plan(mc, N, K, sms > 0 ? sms : 148).ws_bytes;
}

namespace {
bool lmh_shape(int64_t M, int64_t N, int64_t K) {
  if ((g_debug_flags & ~2) != 0) return false;
  const int dev = current_device();
  return dev >= 0 && lmh_eligible(M, N, K, device_sm_count(dev));
}
}  // namespace

extern "C" int ddq_lm_head_argmax(const void* x, const uint8_t* wq, const float* scales, int64_t M,
                                  int64_t N, int64_t K, int64_t vocab_offset, uint64_t* packed,
                                  int64_t* ids, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  if (M < 0 || N < 0 || K < 0 || vocab_offset < 0) return DDQ_ERR_SHAPE;
  if (M == 0) return DDQ_OK;
  if (!x || !packed || (N > 0 && (!wq || !scales))) return DDQ_ERR_INVALID_ARGUMENT;
  if (M > 0x7fffffff || N > 0x7fffffff || vocab_offset + N > 0xFFFFFFFFll) return DDQ_ERR_SHAPE;
  if (!(K > 0 && K % 16 == 0 && K <= 12288 && aligned16(x) && aligned16(wq))) return DDQ_ERR_ALIGNMENT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int dev = current_device();
  const int sms = dev >= 0 ? device_sm_count(dev) : -1;
  const size_t area = lmh_area_bytes(sms);
  if (N > 0 && lmh_shape(M, N, K)) {
    // one streaming kernel writes packed and ids (no memset, split or unpack)
    return launch_lmh(reinterpret_cast<const __half*>(x), wq, scales, (int)M, (int)N, (int)K,
                      vocab_offset, reinterpret_cast<unsigned long long*>(packed), ids, workspace,
                      workspace_bytes, g_wait_timeout_ns, g_debug_flags, s);
  }
  // the decode-kernel path keeps its planes after the streaming kernel's area
  void* dws = nullptr;
  size_t dws_bytes = 0;
  if (workspace && workspace_bytes > area) {
    dws = static_cast<uint8_t*>(workspace) + area;
    dws_bytes = workspace_bytes - area;
  }
  // every chunk on the decode kernel: its split pre-pass zeroes the chunk's
  // packed words, and its last CTA writes the ids (arrival counter at byte 64
  // of the streaming kernel's area, zero between calls); otherwise a memset
  // before and the unpack kernel after
  const int64_t last_mc = M - (M - 1) / kLmChunk * kLmChunk;  // the smallest chunk
  const bool dec_all = N > 0 && last_mc >= tc_min_m();
  unsigned int* counter =
      dec_all && ids && dws ? reinterpret_cast<unsigned int*>(static_cast<uint8_t*>(workspace) + 64)
                            : nullptr;
  if (!dec_all &&
      cudaMemsetAsync(packed, 0, (size_t)M * sizeof(uint64_t), s) != cudaSuccess)
    return DDQ_ERR_LAUNCH;
  if (N > 0) {
    const __half* xh = reinterpret_cast<const __half*>(x);
    unsigned long long* pk = reinterpret_cast<unsigned long long*>(packed);
    for (int64_t m0 = 0; m0 < M; m0 += kLmChunk) {
      const int mc = (int)(M - m0 < kLmChunk ? M - m0 : kLmChunk);
      int st;
      if (mc >= tc_min_m())
        st = launch_dec(xh + m0 * K, wq, scales, nullptr, DDQ_DTYPE_NONE, nullptr, pk + m0,
                        vocab_offset, mc, (int)N, (int)K, dws, dws_bytes,
                        g_wait_timeout_ns, g_debug_flags, s, false, nullptr, nullptr,
                        counter ? ids + m0 : nullptr, counter);
      else
        st = launch_skinny_argmax(xh + m0 * K, wq, scales, pk + m0, vocab_offset, mc, (int)N,
                                  (int)K, s);
      if (st != DDQ_OK) return st;
    }
  }
  if (ids && !counter)
    return launch_unpack_argmax(reinterpret_cast<const unsigned long long*>(packed), M, ids, s);
  return DDQ_OK;
}

extern "C" int ddq_unpack_argmax(const uint64_t* packed, int64_t M, int64_t* ids, void* stream) {
  if (M < 0) return DDQ_ERR_SHAPE;
  if (M == 0) return DDQ_OK;
  if (!packed || !ids) return DDQ_ERR_INVALID_ARGUMENT;
  return launch_unpack_argmax(reinterpret_cast<const unsigned long long*>(packed), M, ids,
                              reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int ddq_set_debug(int flags, uint64_t wait_timeout_ns) {
  if (flags < 0) return DDQ_ERR_INVALID_ARGUMENT;
  g_debug_flags = flags;
  g_wait_timeout_ns = wait_timeout_ns ? wait_timeout_ns : 1000000000ull;
  return DDQ_OK;
}

extern "C" int ddq_read_trace(uint64_t* dst, int max_ctas, void* stream) {
  if (!dst || max_ctas < 0) return DDQ_ERR_INVALID_ARGUMENT;
  const int n = max_ctas < kTraceCtas ? max_ctas : kTraceCtas;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (n > 0 && cudaMemcpyFromSymbolAsync(dst, g_trace, (size_t)n * kTraceSlots * sizeof(uint64_t),
                                         0, cudaMemcpyDeviceToHost, s) != cudaSuccess)
    return DDQ_ERR_LAUNCH;
  if (cudaStreamSynchronize(s) != cudaSuccess) return DDQ_ERR_LAUNCH;
  return DDQ_OK;
}

extern "C" int ddq_device_error(int* code, void* stream) {
  if (!code) return DDQ_ERR_INVALID_ARGUMENT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int zero = 0;
  if (cudaMemcpyFromSymbolAsync(code, g_device_error, sizeof(int), 0, cudaMemcpyDeviceToHost, s) != cudaSuccess)
    return DDQ_ERR_LAUNCH;
  if (cudaMemcpyToSymbolAsync(g_device_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s) != cudaSuccess)
    return DDQ_ERR_LAUNCH;
  if (cudaStreamSynchronize(s) != cudaSuccess) return DDQ_ERR_LAUNCH;
  return DDQ_OK;
}
