// C ABI of libnvfp4_b200.so: plain pointers, sizes and strides; no torch types.
// Declarations and the reference interface each entry point replaces are in
// include/nvfp4_b200.h.
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>

#include "common.cuh"
#include "kernels.h"
#include "../../include/nvfp4_b200.h"

using namespace nvfp4;


static thread_local char g_err[512] = "";

static int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
static int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int nvfp4_record_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

// One device-resident status word per device; kernels record bounded-wait
// timeouts here (0 = ok).
static __device__ int g_status_word;

namespace nvfp4 {
// Address of the status word on `dev` (the current device); nullptr if it
// cannot be looked up.  Shared with the allocation-free GEMV entry point.
int* device_status_word(int dev);
void noalloc_scratch_reset(int dev);
}  // namespace nvfp4

static int* status_ptr(int dev) { return nvfp4::device_status_word(dev); }

int* nvfp4::device_status_word(int dev) {
  static int* ptrs[64] = {nullptr};
  if (dev < 0 || dev >= 64) return nullptr;
  if (!ptrs[dev]) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_status_word) != cudaSuccess) return nullptr;
    ptrs[dev] = static_cast<int*>(p);
  }
  return ptrs[dev];
}

static int num_sms_of(int dev) {
  static int cache[64] = {0};
  if (dev < 0 || dev >= 64) return 148;
  if (!cache[dev]) {
    int n = 0;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    cache[dev] = n > 0 ? n : 148;
  }
  return cache[dev];
}

// Per-device workspaces for kernels that combine partial results across CTAs
// (kind 0: the tensor-core GEMV; kind 1: the stream-K GEMM).  Allocated on the first call that needs it (and
// grown when a later call needs more), zeroed once; the kernels leave it
// zeroed.  Calls on one device share it, so they must not overlap on the GPU.
struct DeviceWorkspace {
  void* ptr = nullptr;
  size_t bytes = 0;
};
enum { kWsGemv = 0, kWsGemm = 1 };
static DeviceWorkspace g_ws[2][64];
static std::mutex g_ws_mutex;

static void* workspace_for(int kind, int dev, size_t bytes, cudaStream_t stream, cudaError_t* err) {
  *err = cudaSuccess;
  if (dev < 0 || dev >= 64) {
    *err = cudaErrorInvalidDevice;
    return nullptr;
  }
  std::lock_guard<std::mutex> lock(g_ws_mutex);
  DeviceWorkspace& w = g_ws[kind][dev];
  if (w.bytes >= bytes) return w.ptr;
  // Growing the workspace synchronises the device and allocates, neither of
  // which a stream capture allows: make one uncaptured call of the largest
  // shape first.
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(stream, &cap) == cudaSuccess && cap != cudaStreamCaptureStatusNone) {
    *err = cudaErrorStreamCaptureUnsupported;
    return nullptr;
  }
  if (w.ptr) {
    // earlier launches may still read the old buffer
    if ((*err = cudaDeviceSynchronize()) != cudaSuccess) return nullptr;
    cudaFree(w.ptr);
    w.ptr = nullptr;
    w.bytes = 0;
  }
  size_t want = bytes < (1u << 20) ? (1u << 20) : bytes;
  if ((*err = cudaMalloc(&w.ptr, want)) != cudaSuccess) return nullptr;
  if ((*err = cudaMemsetAsync(w.ptr, 0, want, stream)) != cudaSuccess) return nullptr;
  w.bytes = want;
  return w.ptr;
}

extern "C" char** environ;

namespace nvfp4 {
EnvOptions read_env_options() {
  EnvOptions o;
  for (char** e = environ; e && *e; ++e) {
    const char* v = *e;
    if (strncmp(v, "NVFP4_", 6) != 0) continue;
    v += 6;
    auto key = [&](const char* k) -> const char* {  // value if v is "k=..."
      const size_t n = strlen(k);
      return (strncmp(v, k, n) == 0 && v[n] == '=') ? v + n + 1 : nullptr;
    };
    const char* x;
    if ((x = key("GEMM_BN"))) o.gemm_bn = atoi(x);
    else if ((x = key("SPLITS"))) o.splits = atoi(x);
    else if ((x = key("PAIR"))) o.pair = (x[0] == '0') ? 0 : (x[0] == '1') ? 1 : -1;
    else if ((x = key("STREAMK"))) o.streamk = atoi(x);
    else if ((x = key("PREFETCH"))) o.prefetch = atoi(x);
    else if ((x = key("FAULT_INJECT"))) o.fault_inject = (x[0] == '1');
    else if ((x = key("GEMV_PATH"))) o.gemv_simt = (strcmp(x, "simt") == 0);
    else if ((x = key("GEMV_CTAS"))) o.gemv_ctas = atoi(x);
    else if ((x = key("B_EVICT"))) o.b_evict = atoi(x);
  }
  return o;
}
}  // namespace nvfp4

static bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

#define NVFP4_API extern "C" __attribute__((visibility("default")))

NVFP4_API const char* nvfp4_last_error(void) { return g_err; }

NVFP4_API int nvfp4_abi_version(void) { return 2; }

NVFP4_API int nvfp4_device_status(int clear) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -1;
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_status_word, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    // A bounded wait ran out: the kernel that gave up may have left arrival
    // counters, stream-K flags or partial sums in the shared workspaces.  Wait
    // for the device, then zero every workspace of this device (and the
    // allocation-free GEMV's scratch) so that the next call starts clean.
    cudaDeviceSynchronize();
    {
      std::lock_guard<std::mutex> lock(g_ws_mutex);
      for (int kind = 0; kind < 2; ++kind)
        if (dev >= 0 && dev < 64 && g_ws[kind][dev].ptr) cudaMemset(g_ws[kind][dev].ptr, 0, g_ws[kind][dev].bytes);
    }
    nvfp4::noalloc_scratch_reset(dev);
    const int zero = 0;
    cudaMemcpyToSymbol(g_status_word, &zero, sizeof(int));
    cudaDeviceSynchronize();
  }
  return v;
}

NVFP4_API int nvfp4_gemv(const void* a, const void* b, const void* sfa_blk, const void* sfb_blk, void* c, int M,
                         int K, int L, int64_t a_lstride, int64_t b_lstride, int64_t sfa_lstride, int64_t sfb_lstride,
                         int64_t c_lstride, void* stream) {
  if (!a || !b || !sfa_blk || !sfb_blk || !c) return fail(NVFP4_ERR_NULL, "nvfp4_gemv: null pointer");
  if (M <= 0 || K <= 0 || L <= 0) return fail(NVFP4_ERR_SHAPE, "nvfp4_gemv: M, K, L must be positive");
  if (M % 128 != 0) return fail(NVFP4_ERR_SHAPE, "nvfp4_gemv: M=%d must be a multiple of 128", M);
  if (K % 64 != 0) return fail(NVFP4_ERR_SHAPE, "nvfp4_gemv: K=%d must be a multiple of 64", K);
  if (!aligned(a, 16) || !aligned(b, 16) || !aligned(sfa_blk, 16) || !aligned(sfb_blk, 16) || !aligned(c, 2) ||
      (a_lstride % 16) || (b_lstride % 16) || (sfa_lstride % 16) || (sfb_lstride % 16))
    return fail(NVFP4_ERR_ALIGN, "nvfp4_gemv: operands and scales need 16-byte aligned bases and batch strides");
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(NVFP4_ERR_DEVICE, "nvfp4_gemv: no CUDA device");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const EnvOptions opt = read_env_options();
  const int ctas = (opt.gemv_ctas > 0 && opt.gemv_ctas < num_sms_of(dev)) ? opt.gemv_ctas : num_sms_of(dev);
  const bool simt = (K % 256 != 0) || opt.gemv_simt || gemv_tc_workspace_bytes(M, K, L, ctas) == 0;
  if (!simt) {
    GemvTcArgs g{};
    g.a = a;
    g.b = b;
    g.sfa = sfa_blk;
    g.sfb = sfb_blk;
    g.c = c;
    g.M = M;
    g.K = K;
    g.L = L;
    g.a_lstride = a_lstride;
    g.b_lstride = b_lstride;
    g.sfa_lstride = sfa_lstride;
    g.sfb_lstride = sfb_lstride;
    g.c_lstride = c_lstride;
    g.workspace_bytes = gemv_tc_workspace_bytes(M, K, L, ctas);
    cudaError_t e = cudaSuccess;
    g.workspace = workspace_for(kWsGemv, dev, g.workspace_bytes, s, &e);
    if (!g.workspace)
      return fail(NVFP4_ERR_CUDA, "nvfp4_gemv: workspace: %s",
                  e == cudaErrorStreamCaptureUnsupported
                      ? "it must grow, which a stream capture does not allow; make one uncaptured call of this shape "
                        "first"
                      : cudaGetErrorString(e));
    g.status = status_ptr(dev);
    g.inject = opt.fault_inject;
    const char* why = nullptr;
    e = launch_gemv_tc(g, ctas, s, &why);
    if (e != cudaSuccess) return fail(NVFP4_ERR_CUDA, "nvfp4_gemv: %s", why ? why : cudaGetErrorString(e));
    return NVFP4_OK;
  }
  GemvParams p;
  p.a = static_cast<const uint8_t*>(a);
  p.b = static_cast<const uint8_t*>(b);
  p.sfa = static_cast<const uint8_t*>(sfa_blk);
  p.sfb = static_cast<const uint8_t*>(sfb_blk);
  p.c = static_cast<__half*>(c);
  p.M = M;
  p.K = K;
  p.L = L;
  p.a_lstride = a_lstride;
  p.b_lstride = b_lstride;
  p.sfa_lstride = sfa_lstride;
  p.sfb_lstride = sfb_lstride;
  p.c_lstride = c_lstride;
  p.ctas_per_l = 1;
  cudaError_t e = launch_gemv(p, num_sms_of(dev), s);
  if (e != cudaSuccess) return fail(NVFP4_ERR_CUDA, "nvfp4_gemv: launch failed: %s", cudaGetErrorString(e));
  return NVFP4_OK;
}

static int check_gemm_common(const char* name, const void* a, const void* b, const void* sfa, const void* sfb,
                             const void* c, int M, int N, int K, int L, int64_t a_lstride, int64_t b_lstride,
                             int64_t sfa_lstride, int64_t sfb_lstride, int64_t ldc, int64_t c_lstride) {
  if (!a || !b || !sfa || !sfb || !c) return fail(NVFP4_ERR_NULL, "%s: null pointer", name);
  if (M <= 0 || N <= 0 || K <= 0 || L <= 0) return fail(NVFP4_ERR_SHAPE, "%s: sizes must be positive", name);
  if (M % 128 || N % 128)
    return fail(NVFP4_ERR_SHAPE, "%s: M=%d and N=%d must be multiples of 128", name, M, N);
  if (K % 64) return fail(NVFP4_ERR_SHAPE, "%s: K=%d must be a multiple of 64", name, K);
  if (ldc < N) return fail(NVFP4_ERR_SHAPE, "%s: ldc=%lld < N=%d", name, (long long)ldc, N);
  if (!aligned(a, 16) || !aligned(b, 16) || !aligned(sfa, 16) || !aligned(sfb, 16) || !aligned(c, 16) ||
      (a_lstride % 16) || (b_lstride % 16) || (sfa_lstride % 16) || (sfb_lstride % 16) || (ldc % 8) ||
      (c_lstride % 8))
    return fail(NVFP4_ERR_ALIGN,
                "%s: operands and scales need 16-byte aligned bases and batch strides; ldc and the C batch "
                "stride must be multiples of 8",
                name);
  return NVFP4_OK;
}

// Copies a GEMM plan into the launch arguments and attaches the stream-K
// workspace when the plan needs one.
static int apply_plan(const char* who, int dev, const GemmPlan& pl, GemmArgs& g, void* stream) {
  g.bn = pl.bn;
  g.splits = pl.splits;
  g.streamk = pl.streamk;
  g.streamk_pure = pl.streamk_pure;
  g.pair = pl.pair;
  if (pl.workspace_bytes) {
    cudaError_t we;
    g.workspace = workspace_for(kWsGemm, dev, pl.workspace_bytes, static_cast<cudaStream_t>(stream), &we);
    if (!g.workspace)
      return fail(NVFP4_ERR_CUDA, "%s: workspace: %s", who,
                  we == cudaErrorStreamCaptureUnsupported
                      ? "it must grow, which a stream capture does not allow; make one uncaptured call of this shape "
                        "first"
                      : cudaGetErrorString(we));
    g.workspace_bytes = pl.workspace_bytes;
  }
  return NVFP4_OK;
}

NVFP4_API int nvfp4_gemm(const void* a, const void* b, const void* sfa_blk, const void* sfb_blk, void* c, int M, int N, int K,
               int L, int64_t a_lstride, int64_t b_lstride, int64_t sfa_lstride, int64_t sfb_lstride, int64_t ldc,
               int64_t c_lstride, void* stream) {
  int rc = check_gemm_common("nvfp4_gemm", a, b, sfa_blk, sfb_blk, c, M, N, K, L, a_lstride, b_lstride, sfa_lstride,
                             sfb_lstride, ldc, c_lstride);
  if (rc) return rc;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(NVFP4_ERR_DEVICE, "nvfp4_gemm: no CUDA device");
  GemmArgs g{};
  g.a = a;
  g.b = b;
  g.b2 = b;
  g.sfa = sfa_blk;
  g.sfb = sfb_blk;
  g.sfb2 = sfb_blk;
  g.c = c;
  g.M = M;
  g.N = N;
  g.K = K;
  g.L = L;
  g.a_lstride = a_lstride;
  g.b_lstride = b_lstride;
  g.b2_lstride = b_lstride;
  g.sfa_lstride = sfa_lstride;
  g.sfb_lstride = sfb_lstride;
  g.sfb2_lstride = sfb_lstride;
  g.ldc = ldc;
  g.c_lstride = c_lstride;
  g.status = status_ptr(dev);
  const EnvOptions opt = read_env_options();
  const GemmPlan pl = gemm_plan(M, N, K, L, false, num_sms_of(dev), opt);
  g.prefetch = opt.prefetch;
  g.inject = opt.fault_inject;
  g.b_evict = opt.b_evict >= 0 ? opt.b_evict : pl.b_evict;
  rc = apply_plan("nvfp4_gemm", dev, pl, g, stream);
  if (rc) return rc;
  const char* why = nullptr;
  cudaError_t e = launch_gemm(g, num_sms_of(dev), static_cast<cudaStream_t>(stream), &why);
  if (e != cudaSuccess)
    return fail(NVFP4_ERR_CUDA, "nvfp4_gemm: %s", why ? why : cudaGetErrorString(e));
  return NVFP4_OK;
}

NVFP4_API int nvfp4_dual_gemm(const void* a, const void* b1, const void* b2, const void* sfa_blk, const void* sfb1_blk,
                    const void* sfb2_blk, void* c, int M, int N, int K, int L, int64_t a_lstride, int64_t b_lstride,
                    int64_t sfa_lstride, int64_t sfb_lstride, int64_t ldc, int64_t c_lstride, void* stream) {
  int rc = check_gemm_common("nvfp4_dual_gemm", a, b1, sfa_blk, sfb1_blk, c, M, N, K, L, a_lstride, b_lstride,
                             sfa_lstride, sfb_lstride, ldc, c_lstride);
  if (rc) return rc;
  if (!b2 || !sfb2_blk) return fail(NVFP4_ERR_NULL, "nvfp4_dual_gemm: null pointer");
  if (!aligned(b2, 16) || !aligned(sfb2_blk, 16))
    return fail(NVFP4_ERR_ALIGN, "nvfp4_dual_gemm: b2 and its scales need 16-byte alignment");
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(NVFP4_ERR_DEVICE, "nvfp4_dual_gemm: no CUDA device");
  GemmArgs g{};
  g.a = a;
  g.b = b1;
  g.b2 = b2;
  g.sfa = sfa_blk;
  g.sfb = sfb1_blk;
  g.sfb2 = sfb2_blk;
  g.c = c;
  g.M = M;
  g.N = N;
  g.K = K;
  g.L = L;
  g.a_lstride = a_lstride;
  g.b_lstride = b_lstride;
  g.b2_lstride = b_lstride;
  g.sfa_lstride = sfa_lstride;
  g.sfb_lstride = sfb_lstride;
  g.sfb2_lstride = sfb_lstride;
  g.ldc = ldc;
  g.c_lstride = c_lstride;
  g.status = status_ptr(dev);
  const EnvOptions opt = read_env_options();
  const GemmPlan pl = gemm_plan(M, N, K, L, true, num_sms_of(dev), opt);
  g.prefetch = opt.prefetch;
  g.inject = opt.fault_inject;
  g.b_evict = opt.b_evict >= 0 ? opt.b_evict : pl.b_evict;
  rc = apply_plan("nvfp4_dual_gemm", dev, pl, g, stream);
  if (rc) return rc;
  const char* why = nullptr;
  cudaError_t e = launch_dual_gemm(g, num_sms_of(dev), static_cast<cudaStream_t>(stream), &why);
  if (e != cudaSuccess)
    return fail(NVFP4_ERR_CUDA, "nvfp4_dual_gemm: %s", why ? why : cudaGetErrorString(e));
  return NVFP4_OK;
}


NVFP4_API int nvfp4_quantize(const void* x, int dtype, void* packed, void* sf_blk, int rows, int K, int L,
                             int64_t x_lstride, int64_t packed_lstride, int64_t sf_lstride, float global_scale,
                             void* stream) {
  if (!x || !packed || !sf_blk) return fail(NVFP4_ERR_NULL, "nvfp4_quantize: null pointer");
  if (dtype != 0 && dtype != 1) return fail(NVFP4_ERR_SHAPE, "nvfp4_quantize: dtype must be 0 (fp16) or 1 (bf16)");
  if (rows <= 0 || K <= 0 || L <= 0 || rows % 128 || K % 64)
    return fail(NVFP4_ERR_SHAPE, "nvfp4_quantize: rows=%d must be a multiple of 128 and K=%d of 64", rows, K);
  if (!(global_scale > 0.f)) return fail(NVFP4_ERR_SHAPE, "nvfp4_quantize: global_scale must be > 0");
  if (!aligned(x, 32) || !aligned(packed, 8) || !aligned(sf_blk, 4) || (x_lstride % 16) || (packed_lstride % 8) ||
      (sf_lstride % 4))
    return fail(NVFP4_ERR_ALIGN, "nvfp4_quantize: x needs 32-byte, packed 8-byte, scales 4-byte alignment");
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(NVFP4_ERR_DEVICE, "nvfp4_quantize: no CUDA device");
  QuantArgs a{x, dtype, packed, sf_blk, rows, K, L, x_lstride, packed_lstride, sf_lstride, global_scale};
  cudaError_t e = launch_quantize(a, num_sms_of(dev), static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(NVFP4_ERR_CUDA, "nvfp4_quantize: %s", cudaGetErrorString(e));
  return NVFP4_OK;
}

static int scale_layout(const char* name, bool to_blocked, const void* src, void* dst, int rows, int sk, int L,
                        int64_t plain_row_stride, int64_t plain_lstride, int64_t blk_lstride, void* stream) {
  if (!src || !dst) return fail(NVFP4_ERR_NULL, "%s: null pointer", name);
  if (rows <= 0 || sk <= 0 || L <= 0 || rows % 128 || sk % 4)
    return fail(NVFP4_ERR_SHAPE, "%s: rows=%d must be a multiple of 128 and K/16=%d of 4", name, rows, sk);
  if (!aligned(src, 4) || !aligned(dst, 4) || (plain_row_stride % 4) || (plain_lstride % 4) || (blk_lstride % 4))
    return fail(NVFP4_ERR_ALIGN, "%s: bases and strides must be multiples of 4 bytes", name);
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(NVFP4_ERR_DEVICE, "%s: no CUDA device", name);
  ScaleLayoutArgs a{src, dst, rows, sk, L, plain_row_stride, plain_lstride, blk_lstride};
  cudaError_t e = launch_scale_layout(a, to_blocked, num_sms_of(dev), static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(NVFP4_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
  return NVFP4_OK;
}

NVFP4_API int nvfp4_scales_to_blocked(const void* plain, void* blk, int rows, int sk, int L, int64_t plain_row_stride,
                                      int64_t plain_lstride, int64_t blk_lstride, void* stream) {
  return scale_layout("nvfp4_scales_to_blocked", true, plain, blk, rows, sk, L, plain_row_stride, plain_lstride,
                      blk_lstride, stream);
}

NVFP4_API int nvfp4_scales_from_blocked(const void* blk, void* plain, int rows, int sk, int L,
                                        int64_t plain_row_stride, int64_t plain_lstride, int64_t blk_lstride,
                                        void* stream) {
  return scale_layout("nvfp4_scales_from_blocked", false, blk, plain, rows, sk, L, plain_row_stride, plain_lstride,
                      blk_lstride, stream);
}

// ------------------------------------------------------------------ MXFP4 and experts
constexpr int kMaxExpertsApi = 1024;
// Sizes of one dimension: the kernels round them up and step past them in 32-bit
// integers, by less than 2^20.
constexpr int64_t kMaxSize = INT32_MAX - (1 << 20);

static int64_t dtype_size(int dtype) { return dtype == 2 ? 4 : 2; }

// The checks that the quantiser and the dequantiser share; fills `a`.
static int mx_quant_args(const char* name, const nvfp4_mx_quant_args* x, bool quantize, MxQuantArgs& a) {
  if (!x) return fail(NVFP4_ERR_NULL, "%s: null argument block", name);
  if (x->dtype < 0 || x->dtype > 2) return fail(NVFP4_ERR_SHAPE, "%s: dtype must be 0 (fp16), 1 (bf16) or 2 (fp32)", name);
  if (x->rows < 0 || x->K <= 0 || x->experts < 1)
    return fail(NVFP4_ERR_SHAPE, "%s: rows=%d must not be negative, K=%d and experts=%d must be positive", name, x->rows,
                x->K, x->experts);
  if (x->columns && (!quantize || x->offsets || x->slots || x->experts != 1))
    return fail(NVFP4_ERR_SHAPE, "%s: blocks down the columns are for one matrix to be quantised", name);
  if (!x->columns && x->K % 32) return fail(NVFP4_ERR_SHAPE, "%s: K=%d must be a multiple of 32", name, x->K);
  if (x->offsets && x->experts > kMaxExpertsApi)
    return fail(NVFP4_ERR_SHAPE, "%s: %d experts, at most %d", name, x->experts, kMaxExpertsApi);
  if (x->slots && (!quantize || !x->offsets || x->top < 0))
    return fail(NVFP4_ERR_SHAPE, "%s: slots need offsets and top >= 0", name);
  const int64_t rows = x->offsets ? x->rows : static_cast<int64_t>(x->rows) * x->experts;
  const int64_t units = rows * ((static_cast<int64_t>(x->K) + 127) / 128 * 4);  // scales, padding included
  const int64_t sorted = x->slots ? static_cast<int64_t>(x->rows) * x->top : rows;
  if (rows > kMaxSize || x->K > kMaxSize || units > kMaxSize || sorted > kMaxSize ||
      (x->columns && x->rows > 65535 * 256))
    return fail(NVFP4_ERR_SHAPE, "%s: too large", name);
  if (rows > 0 && sorted > 0) {
    if (!x->x || !x->packed || !x->scales) return fail(NVFP4_ERR_NULL, "%s: null pointer", name);
    if (!aligned(x->x, quantize ? dtype_size(x->dtype) : 32) || !aligned(x->packed, 16) || !aligned(x->scales, 16) ||
        !aligned(x->offsets, 4) || !aligned(x->slots, 4))
      return fail(NVFP4_ERR_ALIGN, "%s: codes and scales need 16-byte alignment, x that of its type%s", name,
                  quantize ? "" : " and 32 bytes");
  }
  a = MxQuantArgs{x->x,       x->packed, x->scales, x->offsets, x->slots, x->dtype, static_cast<int>(rows), x->K, x->rows,
                  x->experts, x->top,    static_cast<int>(sorted), x->columns, x->x_rstride, x->x_estride};
  return NVFP4_OK;
}

NVFP4_API int nvfp4_mx_quantize(const nvfp4_mx_quant_args* x) {
  MxQuantArgs a;
  const int rc = mx_quant_args("nvfp4_mx_quantize", x, true, a);
  if (rc) return rc;
  if (a.rows == 0 || a.sorted_rows == 0) return NVFP4_OK;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(NVFP4_ERR_DEVICE, "nvfp4_mx_quantize: no CUDA device");
  const cudaError_t e = launch_mx_quantize(a, num_sms_of(dev), static_cast<cudaStream_t>(x->stream));
  if (e != cudaSuccess) return fail(NVFP4_ERR_CUDA, "nvfp4_mx_quantize: %s", cudaGetErrorString(e));
  return NVFP4_OK;
}

NVFP4_API int nvfp4_mx_dequantize(const nvfp4_mx_quant_args* x) {
  MxQuantArgs a;
  const int rc = mx_quant_args("nvfp4_mx_dequantize", x, false, a);
  if (rc) return rc;
  if (a.rows == 0) return NVFP4_OK;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(NVFP4_ERR_DEVICE, "nvfp4_mx_dequantize: no CUDA device");
  const cudaError_t e = launch_mx_dequantize(a, num_sms_of(dev), static_cast<cudaStream_t>(x->stream));
  if (e != cudaSuccess) return fail(NVFP4_ERR_CUDA, "nvfp4_mx_dequantize: %s", cudaGetErrorString(e));
  return NVFP4_OK;
}

// The checks of a product's sizes.
static int mx_gemm_sizes(const char* name, const nvfp4_mx_gemm_args* x) {
  if (!x) return fail(NVFP4_ERR_NULL, "%s: null argument block", name);
  if (x->out_dtype < 0 || x->out_dtype > 3)
    return fail(NVFP4_ERR_SHAPE, "%s: out_dtype must be 0 (fp16), 1 (bf16), 2 (fp32) or 3 (MXFP4)", name);
  const bool codes = x->out_dtype == 3;
  if (x->rows < 0 || x->N <= 0 || x->K <= 0 || x->experts < 1)
    return fail(NVFP4_ERR_SHAPE, "%s: rows must not be negative; N, K and experts must be positive", name);
  if (x->K % 32) return fail(NVFP4_ERR_SHAPE, "%s: K=%d must be a multiple of 32", name, x->K);
  if (x->experts > kMaxExpertsApi)
    return fail(NVFP4_ERR_SHAPE, "%s: %d experts, at most %d", name, x->experts, kMaxExpertsApi);
  if (x->experts != 1 && !x->offsets) return fail(NVFP4_ERR_NULL, "%s: several experts need offsets", name);
  if (!codes && x->ldc < x->N)
    return fail(NVFP4_ERR_SHAPE, "%s: ldc=%lld < N=%d", name, (long long)x->ldc, x->N);
  if (codes && (x->N % 32 || !x->b2))
    return fail(NVFP4_ERR_SHAPE, "%s: an MXFP4 result is for two products, N=%d a multiple of 32", name, x->N);
  if (x->rows > kMaxSize || x->N > kMaxSize || x->K > (1 << 24) ||
      (static_cast<int64_t>(x->rows) / 32 + x->experts) * ((static_cast<int64_t>(x->N) + 63) / 64) > kMaxSize)
    return fail(NVFP4_ERR_SHAPE, "%s: too large", name);
  return NVFP4_OK;
}

NVFP4_API int nvfp4_mx_gemm(const nvfp4_mx_gemm_args* x) {
  const char* name = "nvfp4_mx_gemm";
  const int rc = mx_gemm_sizes(name, x);
  if (rc) return rc;
  const bool codes = x->out_dtype == 3;
  if (x->rows == 0) return NVFP4_OK;
  if (!x->a || !x->b || !x->sfa || !x->sfb || !x->c || !x->b2 != !x->sfb2 || (codes && !x->c_scales))
    return fail(NVFP4_ERR_NULL, "%s: null pointer", name);
  if (!aligned(x->a, 16) || !aligned(x->b, 16) || !aligned(x->b2, 16) || !aligned(x->sfa, 16) || !aligned(x->sfb, 16) ||
      !aligned(x->sfb2, 16) || !aligned(x->c, codes ? 16 : dtype_size(x->out_dtype)) || !aligned(x->c_scales, 16) ||
      !aligned(x->offsets, 4))
    return fail(NVFP4_ERR_ALIGN, "%s: codes and scales need 16-byte alignment, c that of its type", name);
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(NVFP4_ERR_DEVICE, "%s: no CUDA device", name);
  MxGemmArgs g{x->a,    x->b, x->b2, x->sfa,     x->sfb,       x->sfb2, x->c, x->c_scales, x->offsets,
               x->rows, x->N, x->K,  x->experts, x->out_dtype, x->ldc,  status_ptr(dev), read_env_options().fault_inject};
  const char* why = nullptr;
  const cudaError_t e = launch_mx_gemm(g, num_sms_of(dev), static_cast<cudaStream_t>(x->stream), &why);
  if (e != cudaSuccess) return fail(NVFP4_ERR_CUDA, "%s: %s", name, why ? why : cudaGetErrorString(e));
  return NVFP4_OK;
}

NVFP4_API int nvfp4_mx_gemm_shape(const nvfp4_mx_gemm_args* x, int num_sms, int32_t* tokens, int32_t* ctas,
                                  int32_t* k_splits) {
  const char* name = "nvfp4_mx_gemm_shape";
  const int rc = mx_gemm_sizes(name, x);
  if (rc) return rc;
  if (x->rows == 0 || num_sms < 2) return fail(NVFP4_ERR_SHAPE, "%s: rows must be positive, num_sms 2 or more", name);
  if (!tokens || !ctas || !k_splits) return fail(NVFP4_ERR_NULL, "%s: null pointer", name);
  MxGemmArgs g{};
  g.b2 = x->b2;
  g.offsets = x->offsets;
  g.rows = x->rows;
  g.N = x->N;
  g.K = x->K;
  g.experts = x->experts;
  const MxGemmShape shape = mx_gemm_shape(g, num_sms);
  *tokens = shape.tn;
  *ctas = shape.pair ? 2 : 1;
  *k_splits = shape.splits;
  return NVFP4_OK;
}

NVFP4_API int64_t nvfp4_moe_sort_workspace(int n, int experts) {
  int dev = 0;
  if (n < 0 || n > kMaxSize || experts < 1 || experts > kMaxExpertsApi || cudaGetDevice(&dev) != cudaSuccess) return -1;
  return static_cast<int64_t>(moe_sort_workspace_bytes(n, experts, num_sms_of(dev)));
}

NVFP4_API int nvfp4_moe_sort(const void* ids, int id_bytes, int n, int experts, int32_t* order, int32_t* slots,
                             int32_t* offsets, void* workspace, int64_t workspace_bytes, void* stream) {
  if (id_bytes != 4 && id_bytes != 8) return fail(NVFP4_ERR_SHAPE, "nvfp4_moe_sort: ids must have 4 or 8 bytes");
  if (n < 0 || n > kMaxSize)
    return fail(NVFP4_ERR_SHAPE, "nvfp4_moe_sort: n=%d must be 0 to %lld", n, (long long)kMaxSize);
  if (experts < 1 || experts > kMaxExpertsApi)
    return fail(NVFP4_ERR_SHAPE, "nvfp4_moe_sort: experts=%d must be 1 to %d", experts, kMaxExpertsApi);
  if (!offsets || (n && (!ids || !order || !slots))) return fail(NVFP4_ERR_NULL, "nvfp4_moe_sort: null pointer");
  if (!aligned(ids, id_bytes) || !aligned(order, 4) || !aligned(slots, 4) || !aligned(offsets, 4) ||
      !aligned(workspace, 4))
    return fail(NVFP4_ERR_ALIGN, "nvfp4_moe_sort: every pointer needs its type's alignment");
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(NVFP4_ERR_DEVICE, "nvfp4_moe_sort: no CUDA device");
  const size_t need = moe_sort_workspace_bytes(n, experts, num_sms_of(dev));
  if (need && (!workspace || workspace_bytes < static_cast<int64_t>(need)))
    return fail(NVFP4_ERR_SHAPE, "nvfp4_moe_sort: the workspace needs %zu bytes", need);
  MoeSortArgs a{ids, id_bytes, n, experts, order, slots, offsets, static_cast<int*>(workspace), 0};
  const cudaError_t e = launch_moe_sort(a, num_sms_of(dev), static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(NVFP4_ERR_CUDA, "nvfp4_moe_sort: %s", cudaGetErrorString(e));
  return NVFP4_OK;
}

static int moe_rows(const char* name, MoeRowOp op, const nvfp4_moe_args* x) {
  if (!x) return fail(NVFP4_ERR_NULL, "%s: null argument block", name);
  if (x->dtype < 0 || x->dtype > 2) return fail(NVFP4_ERR_SHAPE, "%s: dtype must be 0 (fp16), 1 (bf16) or 2 (fp32)", name);
  if (x->tokens < 0 || x->top < 0 || x->hidden < 0 || x->experts < 1 || x->experts > kMaxExpertsApi)
    return fail(NVFP4_ERR_SHAPE, "%s: tokens, top and hidden must not be negative, experts=%d must be 1 to %d", name,
                x->experts, kMaxExpertsApi);
  if (x->tokens > kMaxSize || static_cast<int64_t>(x->tokens) * x->top > kMaxSize || x->hidden > kMaxSize)
    return fail(NVFP4_ERR_SHAPE, "%s: too large", name);
  const bool weighted = op == kMoeCombine || op == kMoeCombineBackward;
  const bool sorted_out = op == kMoeGather || op == kMoeCombineBackward;
  const bool any = x->tokens && x->hidden;   // something to write by token
  const bool rows = x->tokens && x->top;     // something to read or write by row
  if ((any && !x->out && !(sorted_out && !rows)) || (any && rows && !x->in) || (rows && !x->slots) ||
      (rows && sorted_out && !x->offsets) || (rows && weighted && !x->weights) ||
      (rows && op == kMoeCombineBackward && (!x->dweights || (any && !x->grad))))
    return fail(NVFP4_ERR_NULL, "%s: null pointer", name);
  const int64_t size = dtype_size(x->dtype);
  if (!aligned(x->in, size) || !aligned(x->out, size) || !aligned(x->grad, size) || !aligned(x->slots, 4) ||
      !aligned(x->offsets, 4) || !aligned(x->weights, 4) || !aligned(x->dweights, 4))
    return fail(NVFP4_ERR_ALIGN, "%s: every pointer needs its type's alignment", name);
  if (!x->tokens || (!x->hidden && op != kMoeCombineBackward) || (sorted_out && !x->top)) return NVFP4_OK;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(NVFP4_ERR_DEVICE, "%s: no CUDA device", name);
  MoeRowArgs a{x->in,    x->grad, x->weights, x->out,    x->dweights, x->slots,     x->offsets,
               x->dtype, x->tokens, x->top,   x->hidden, x->experts,  x->in_stride, x->grad_stride};
  const cudaError_t e = launch_moe_rows(op, a, num_sms_of(dev), static_cast<cudaStream_t>(x->stream));
  if (e != cudaSuccess) return fail(NVFP4_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
  return NVFP4_OK;
}

NVFP4_API int nvfp4_moe_gather(const nvfp4_moe_args* x) { return moe_rows("nvfp4_moe_gather", kMoeGather, x); }
NVFP4_API int nvfp4_moe_gather_backward(const nvfp4_moe_args* x) {
  return moe_rows("nvfp4_moe_gather_backward", kMoeGatherBackward, x);
}
NVFP4_API int nvfp4_moe_combine(const nvfp4_moe_args* x) { return moe_rows("nvfp4_moe_combine", kMoeCombine, x); }
NVFP4_API int nvfp4_moe_combine_backward(const nvfp4_moe_args* x) {
  return moe_rows("nvfp4_moe_combine_backward", kMoeCombineBackward, x);
}

// Packed-argument forms (include/nvfp4_b200.h): the same calls, one pointer.
NVFP4_API int nvfp4_gemv_call(const nvfp4_gemv_args* x) {
  if (!x) return fail(NVFP4_ERR_NULL, "nvfp4_gemv_call: null argument block");
  return nvfp4_gemv(x->a, x->b, x->sfa_blk, x->sfb_blk, x->c, x->M, x->K, x->L, x->a_lstride, x->b_lstride,
                    x->sfa_lstride, x->sfb_lstride, x->c_lstride, x->stream);
}

NVFP4_API int nvfp4_gemm_call(const nvfp4_gemm_args* x) {
  if (!x) return fail(NVFP4_ERR_NULL, "nvfp4_gemm_call: null argument block");
  return nvfp4_gemm(x->a, x->b, x->sfa_blk, x->sfb_blk, x->c, x->M, x->N, x->K, x->L, x->a_lstride, x->b_lstride,
                    x->sfa_lstride, x->sfb_lstride, x->ldc, x->c_lstride, x->stream);
}

NVFP4_API int nvfp4_dual_gemm_call(const nvfp4_gemm_args* x) {
  if (!x) return fail(NVFP4_ERR_NULL, "nvfp4_dual_gemm_call: null argument block");
  return nvfp4_dual_gemm(x->a, x->b, x->b2, x->sfa_blk, x->sfb_blk, x->sfb2_blk, x->c, x->M, x->N, x->K, x->L,
                         x->a_lstride, x->b_lstride, x->sfa_lstride, x->sfb_lstride, x->ldc, x->c_lstride, x->stream);
}
