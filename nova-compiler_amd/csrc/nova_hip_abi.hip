// C ABI of libnova_hip: descriptor validation, flag decoding, per-thread
// stream and error text, and the per-stream workspace cache.  Every check
// here runs on the host before any HIP call, so malformed calls fail with a
// status code instead of reaching a kernel.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>
#include <memory>
#include <numeric>
#include <unordered_map>
#include <vector>

#include "nova_hip_internal.h"

namespace nova_hip {

namespace {
thread_local char t_err[512] = {0};
thread_local hipStream_t t_stream = nullptr;

struct Workspace {
  void *ptr = nullptr;
  size_t bytes = 0;
};
std::mutex g_ws_mu;
std::unordered_map<hipStream_t, Workspace> g_ws;

// One enqueue mutex per stream, never erased (a later stream with a
// recycled handle shares it, which only serialises more).  Lock order: a
// stream's mutex, then g_ws_mu.
std::mutex g_stream_mu_mu;
std::unordered_map<hipStream_t, std::unique_ptr<std::mutex>> g_stream_mu;

std::mutex &stream_mutex(hipStream_t s) {
  std::lock_guard<std::mutex> lock(g_stream_mu_mu);
  std::unique_ptr<std::mutex> &m = g_stream_mu[s];
  if (!m) m.reset(new std::mutex);
  return *m;
}
}  // namespace

int32_t fail(int32_t code, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(t_err, sizeof(t_err), fmt, ap);
  va_end(ap);
  return code;
}

void clear_error() { t_err[0] = 0; }

hipStream_t current_stream() { return t_stream; }

namespace {
// A device attribute of the current device, queried once per device.
int cached_attribute(std::atomic<int> *cache, int n, hipDeviceAttribute_t attr) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0) return 0;
  if (dev < n) {
    const int c = cache[dev].load(std::memory_order_relaxed);  // 0: not queried yet
    if (c) return c > 0 ? c : 0;
  }
  int v = 0;
  if (hipDeviceGetAttribute(&v, attr, dev) != hipSuccess) v = 0;
  if (dev < n) cache[dev].store(v > 0 ? v : -1, std::memory_order_relaxed);
  return v > 0 ? v : 0;
}
constexpr int kMaxDevices = 64;
}  // namespace

int device_cu_count() {
  static std::atomic<int> cache[kMaxDevices];
  return cached_attribute(cache, kMaxDevices, hipDeviceAttributeMultiprocessorCount);
}

int device_lds_per_block() {
  static std::atomic<int> cache[kMaxDevices];
  return cached_attribute(cache, kMaxDevices, hipDeviceAttributeMaxSharedMemoryPerBlock);
}

int32_t check_hip(hipError_t e, const char *what) {
  if (e == hipSuccess) return NOVA_HIP_SUCCESS;
  return fail(NOVA_HIP_EDEVICE, "%s: %s", what, hipGetErrorString(e));
}

namespace {
// The stream's buffer, grown to at least `bytes`; the caller holds the
// stream's mutex.
void *workspace_locked(hipStream_t s, size_t bytes) {
  std::lock_guard<std::mutex> lock(g_ws_mu);
  Workspace &w = g_ws[s];
  if (w.bytes >= bytes && w.ptr) return w.ptr;
  if (w.ptr) {
    // The old buffer may still be read by queued work on this stream.
    hipError_t e = hipStreamSynchronize(s);
    if (e != hipSuccess) {
      check_hip(e, "workspace: stream synchronize");
      return nullptr;
    }
    (void)hipFree(w.ptr);
    w.ptr = nullptr;
    w.bytes = 0;
  }
  size_t want = bytes < (1u << 20) ? (1u << 20) : bytes;
  void *p = nullptr;
  hipError_t e = hipMalloc(&p, want);
  if (e != hipSuccess) {
    fail(NOVA_HIP_ENOMEM, "workspace: hipMalloc(%zu): %s", want, hipGetErrorString(e));
    return nullptr;
  }
  w.ptr = p;
  w.bytes = want;
  return p;
}
}  // namespace

void *WorkspaceLease::acquire(hipStream_t s, size_t bytes) {
  lock_ = std::unique_lock<std::mutex>(stream_mutex(s));
  ptr_ = workspace_locked(s, bytes);
  return ptr_;
}

bool WorkspaceLease::refused_by_capture(hipStream_t s, size_t bytes) {
  {
    std::lock_guard<std::mutex> lock(g_ws_mu);
    const auto it = g_ws.find(s);
    if (it != g_ws.end() && it->second.ptr && it->second.bytes >= bytes) return false;
  }
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(s, &status) != hipSuccess) {
    (void)hipGetLastError();
    return false;
  }
  return status != hipStreamCaptureStatusNone;
}

namespace {

// ---- descriptor helpers ----------------------------------------------------
template <typename D>
const char *data_of(const D *d) {
  return static_cast<const char *>(d->aligned);
}

template <typename D>
bool nonneg_sizes(const D *d, int rank) {
  for (int i = 0; i < rank; ++i)
    if (d->sizes[i] < 0) return false;
  return true;
}

int decode_flags(int32_t flags, int &in_dt, int &out_dt, int &epi, int &bias_dt) {
  if (flags & ~(0xffff | NOVA_HIP_GEMM_ACC_OUT | NOVA_HIP_GEMM_F32_MFMA | NOVA_HIP_GEMM_ACC_C))
    return fail(NOVA_HIP_EINVAL, "gemm: unknown flag bits 0x%x", flags);
  in_dt = flags & 0xf;
  out_dt = (flags >> 4) & 0xf;
  epi = (flags >> 8) & 0xf;
  bias_dt = (flags >> 12) & 0xf;
  if (in_dt > NOVA_HIP_DT_F16 || out_dt > NOVA_HIP_DT_F16 || bias_dt > NOVA_HIP_DT_F16 ||
      epi > NOVA_HIP_EPI_GELU)
    return fail(NOVA_HIP_EDTYPE, "gemm: bad dtype/epilogue code in flags 0x%x", flags);
  if (in_dt == NOVA_HIP_DT_F32 && out_dt != NOVA_HIP_DT_F32)
    return fail(NOVA_HIP_EDTYPE, "gemm: f32 inputs produce f32 output only");
  if ((flags & NOVA_HIP_GEMM_F32_MFMA) && (in_dt != NOVA_HIP_DT_F32 || (flags & NOVA_HIP_GEMM_ACC_OUT)))
    return fail(NOVA_HIP_EDTYPE, "gemm: the f32 MFMA form takes f32 operands");
  if (flags & NOVA_HIP_GEMM_ACC_OUT) {
    if (in_dt == NOVA_HIP_DT_F32 || out_dt != in_dt)
      return fail(NOVA_HIP_EDTYPE,
                  "gemm: accumulating in the output dtype needs bf16 or f16 inputs of that dtype");
    if (epi == NOVA_HIP_EPI_GELU || epi == NOVA_HIP_EPI_BIAS_GELU ||
        (epi == NOVA_HIP_EPI_BIAS && bias_dt != out_dt))
      return fail(NOVA_HIP_EDTYPE,
                  "gemm: a bf16 / f16 accumulator takes no GELU, and a bias of its own dtype only");
  }
  if (flags & NOVA_HIP_GEMM_ACC_C) {
    // Accumulating into C's data runs on the exact kernel: f32, or a 16-bit
    // accumulator of the operands' own type.
    if (flags & NOVA_HIP_GEMM_F32_MFMA)
      return fail(NOVA_HIP_EINVAL, "gemm: accumulating into C is not an f32 MFMA form");
    if (in_dt != NOVA_HIP_DT_F32 && !(flags & NOVA_HIP_GEMM_ACC_OUT))
      return fail(NOVA_HIP_EDTYPE,
                  "gemm: accumulating into C needs f32 operands, or 16-bit ones with "
                  "NOVA_HIP_GEMM_ACC_OUT");
    if (epi != NOVA_HIP_EPI_NONE)
      return fail(NOVA_HIP_EINVAL, "gemm: accumulating into C takes no epilogue");
  }
  return NOVA_HIP_SUCCESS;
}

// Validate and normalise a batched GEMM given 3-D views, then launch it
// (with launch false: validate only, so that an entry point with several
// outputs can check them all before it writes any).
int32_t gemm_core(const NovaMemRef3D *A, const NovaMemRef3D *B, NovaMemRef3D *C,
                  const NovaMemRef1D *bias, int32_t flags, bool launch = true) {
  clear_error();
  if (!A || !B || !C) return fail(NOVA_HIP_EINVAL, "gemm: null descriptor");
  int in_dt, out_dt, epi, bias_dt;
  int32_t rc = decode_flags(flags, in_dt, out_dt, epi, bias_dt);
  if (rc) return rc;
  if (!nonneg_sizes(A, 3) || !nonneg_sizes(B, 3) || !nonneg_sizes(C, 3))
    return fail(NOVA_HIP_ESHAPE, "gemm: negative size");
  const int64_t batch = C->sizes[0], M = C->sizes[1], N = C->sizes[2];
  const int64_t K = A->sizes[2];
  if (A->sizes[1] != M || B->sizes[2] != N || B->sizes[1] != K)
    return fail(NOVA_HIP_ESHAPE,
                "gemm: shapes A[%lld,%lld,%lld] B[%lld,%lld,%lld] C[%lld,%lld,%lld] disagree",
                (long long)A->sizes[0], (long long)A->sizes[1], (long long)A->sizes[2],
                (long long)B->sizes[0], (long long)B->sizes[1], (long long)B->sizes[2],
                (long long)batch, (long long)M, (long long)N);
  // Batch: equal, or 1 with any stride (broadcast a rank-2 operand).
  if ((A->sizes[0] != batch && A->sizes[0] != 1) || (B->sizes[0] != batch && B->sizes[0] != 1))
    return fail(NOVA_HIP_ESHAPE, "gemm: batch sizes %lld/%lld do not broadcast to %lld",
                (long long)A->sizes[0], (long long)B->sizes[0], (long long)batch);
  const bool has_bias = (epi == NOVA_HIP_EPI_BIAS || epi == NOVA_HIP_EPI_BIAS_GELU);
  if (has_bias) {
    if (!bias || !bias->aligned) return fail(NOVA_HIP_EINVAL, "gemm: epilogue needs a bias");
    if (bias->sizes[0] != N) return fail(NOVA_HIP_ESHAPE, "gemm: bias size %lld != N %lld",
                                         (long long)bias->sizes[0], (long long)N);
    if (bias->strides[0] != 1 && N > 1) return fail(NOVA_HIP_ESTRIDE, "gemm: bias must be contiguous");
  }
  const bool empty = batch == 0 || M == 0 || N == 0;
  // With K == 0 the operands hold no elements (their data pointer may be
  // null) and C is just the epilogue of a zero accumulator.
  if (!empty && (!C->aligned || (K > 0 && (!A->aligned || !B->aligned))))
    return fail(NOVA_HIP_EINVAL, "gemm: null data pointer");

  GemmProblem p;
  p.batch = batch;
  p.M = M;
  p.N = N;
  p.K = K;
  p.in_dt = in_dt;
  p.out_dt = out_dt;
  p.epi = epi;
  p.bias_dt = bias_dt;
  p.acc_out = (flags & NOVA_HIP_GEMM_ACC_OUT) != 0;
  p.f32_mfma = (flags & NOVA_HIP_GEMM_F32_MFMA) != 0;
  p.acc_c = (flags & NOVA_HIP_GEMM_ACC_C) != 0;
  const int esz = dtype_size(in_dt);
  const int osz = dtype_size(out_dt);
  p.A = data_of(A) + A->offset * esz;
  p.B = data_of(B) + B->offset * esz;
  p.C = const_cast<char *>(data_of(C)) + C->offset * osz;
  p.bias = has_bias ? (const void *)(data_of(bias) + bias->offset * dtype_size(bias_dt)) : nullptr;

  // Each operand is addressed as (unit-stride dim, stride of the other dim).
  // A [M,K]: unit stride on K (row-major) or on M (transposed view).  A
  // dim of extent 1 is never stepped, so its stride does not matter.
  const int64_t a_sm = A->strides[1], a_sk = A->strides[2];
  if (a_sk == 1 || K <= 1) {
    p.a_kcontig = true;
    p.sa_outer = a_sm;
  } else if (a_sm == 1 || M <= 1) {
    p.a_kcontig = false;
    p.sa_outer = a_sk;
  } else {
    return fail(NOVA_HIP_ESTRIDE, "gemm: A strides [%lld,%lld] have no unit stride",
                (long long)a_sm, (long long)a_sk);
  }
  // B [K,N]: unit stride on N (row-major) or on K (transposed view, e.g.
  // nova.transpose of a row-major [N,K] weight).
  const int64_t b_sk = B->strides[1], b_sn = B->strides[2];
  if (b_sn == 1 || N <= 1) {
    p.b_kcontig = false;
    p.sb_outer = b_sk;
  } else if (b_sk == 1 || K <= 1) {
    p.b_kcontig = true;
    p.sb_outer = b_sn;
  } else {
    return fail(NOVA_HIP_ESTRIDE, "gemm: B strides [%lld,%lld] have no unit stride",
                (long long)b_sk, (long long)b_sn);
  }
  if (C->strides[2] != 1 && N > 1) return fail(NOVA_HIP_ESTRIDE, "gemm: C must have unit stride on N");
  if (M > 1 && C->strides[1] < N) return fail(NOVA_HIP_ESTRIDE, "gemm: C rows overlap");
  if (p.sa_outer < 0 || p.sb_outer < 0 || C->strides[1] < 0)
    return fail(NOVA_HIP_ESTRIDE, "gemm: negative strides are not addressed");
  p.sab = (A->sizes[0] == 1) ? 0 : A->strides[0];
  p.sbb = (B->sizes[0] == 1) ? 0 : B->strides[0];
  p.scb = C->strides[0];
  p.scm = C->strides[1];
  if (p.sab < 0 || p.sbb < 0 || p.scb < 0)
    return fail(NOVA_HIP_ESTRIDE, "gemm: negative batch stride");
  if (empty || !launch) return NOVA_HIP_SUCCESS;

  hipStream_t s = current_stream();
  if (p.f32_mfma) {
    // An operand slice beyond the 32-bit buffer range takes the exact kernel.
    rc = launch_gemm_f32_mfma(p, s);
    if (rc != NOVA_HIP_ERANGE) return rc;
    clear_error();
  }
  return (in_dt == NOVA_HIP_DT_F32 || p.acc_out) ? launch_gemm_exact(p, s) : launch_gemm_mfma(p, s);
}

NovaMemRef3D lift(const NovaMemRef2D *d) {
  NovaMemRef3D r;
  r.allocated = d->allocated;
  r.aligned = d->aligned;
  r.offset = d->offset;
  r.sizes[0] = 1;
  r.sizes[1] = d->sizes[0];
  r.sizes[2] = d->sizes[1];
  r.strides[0] = 0;
  r.strides[1] = d->strides[0];
  r.strides[2] = d->strides[1];
  return r;
}

int32_t gemm2d(const NovaMemRef2D *A, const NovaMemRef2D *B, NovaMemRef2D *C,
               const NovaMemRef1D *bias, int32_t flags, bool launch = true) {
  if (!A || !B || !C) {
    clear_error();
    return fail(NOVA_HIP_EINVAL, "gemm: null descriptor");
  }
  NovaMemRef3D a = lift(A), b = lift(B), c = lift(C);
  return gemm_core(&a, &b, &c, bias, flags, launch);
}

NovaMemRef2D transposed(const NovaMemRef2D *d) {
  NovaMemRef2D r = *d;
  r.sizes[0] = d->sizes[1];
  r.sizes[1] = d->sizes[0];
  r.strides[0] = d->strides[1];
  r.strides[1] = d->strides[0];
  return r;
}

// C = A . B into C as laid out: row-major C directly; a transposed view of
// a row-major buffer (unit stride on dim 0) as C^T = B^T . A^T into that
// buffer, since the kernels store rows with unit stride.
int32_t gemm2d_to(const NovaMemRef2D *A, const NovaMemRef2D *B, NovaMemRef2D *C, int32_t flags,
                  bool launch = true) {
  if (C && C->strides[1] != 1 && C->sizes[1] > 1 && (C->strides[0] == 1 || C->sizes[0] <= 1)) {
    NovaMemRef2D at = transposed(A), bt = transposed(B), ct = transposed(C);
    return gemm2d(&bt, &at, &ct, nullptr, flags, launch);
  }
  return gemm2d(A, B, C, nullptr, flags, launch);
}

// Flags of the backward GEMM entry points: dtypes only, no epilogue.
int32_t backward_flags(int32_t flags, int &in_dt, int &out_dt, const char *what) {
  if (flags & (NOVA_HIP_GEMM_ACC_OUT | NOVA_HIP_GEMM_ACC_C))
    return fail(NOVA_HIP_EINVAL, "%s: no narrow-accumulator or accumulate-into form (flags 0x%x)",
                what, flags);
  int epi, bias_dt;
  int32_t rc = decode_flags(flags, in_dt, out_dt, epi, bias_dt);
  if (rc) return rc;
  if (epi != NOVA_HIP_EPI_NONE)
    return fail(NOVA_HIP_EINVAL, "%s: flags carry an epilogue (0x%x)", what, flags);
  return NOVA_HIP_SUCCESS;
}

// Shared validation of the SCE forward entry points (optional softmax and
// fused gradient outputs).
int32_t sce_common(const NovaMemRef2D *logits, const NovaMemRef1D *labels, NovaMemRef1D *loss,
                   NovaMemRef2D *softmax, NovaMemRef2D *grad, const char *what,
                   bool noalloc = false) {
  clear_error();
  if (!logits || !labels || !loss) return fail(NOVA_HIP_EINVAL, "%s: null descriptor", what);
  const int64_t R = logits->sizes[0], C = logits->sizes[1];
  if (R < 0 || C < 0) return fail(NOVA_HIP_ESHAPE, "%s: negative size", what);
  if (labels->sizes[0] != R) return fail(NOVA_HIP_ESHAPE, "%s: labels size != rows", what);
  if (loss->sizes[0] != 1) return fail(NOVA_HIP_ESHAPE, "%s: loss must have shape [1]", what);
  if (softmax && (softmax->sizes[0] != R || softmax->sizes[1] != C))
    return fail(NOVA_HIP_ESHAPE, "%s: softmax shape differs from logits", what);
  if (grad && (grad->sizes[0] != R || grad->sizes[1] != C))
    return fail(NOVA_HIP_ESHAPE, "%s: grad shape differs from logits", what);
  if (C == 0 && R > 0) return fail(NOVA_HIP_ESHAPE, "%s: zero classes", what);
  if ((logits->strides[1] != 1 && C > 1) || (labels->strides[0] != 1 && R > 1) ||
      (softmax && softmax->strides[1] != 1 && C > 1) || (grad && grad->strides[1] != 1 && C > 1))
    return fail(NOVA_HIP_ESTRIDE, "%s: last dim must be contiguous", what);
  if (R > 1 && (logits->strides[0] < C || (softmax && softmax->strides[0] < C) ||
                (grad && grad->strides[0] < C)))
    return fail(NOVA_HIP_ESTRIDE, "%s: rows overlap", what);
  if (!loss->aligned || (R > 0 && (!logits->aligned || !labels->aligned)) ||
      (softmax && !softmax->aligned) || (grad && !grad->aligned))
    return fail(NOVA_HIP_EINVAL, "%s: null data pointer", what);
  SceProblem p;
  p.logits = reinterpret_cast<const float *>(data_of(logits)) + logits->offset;
  p.labels = reinterpret_cast<const int32_t *>(data_of(labels)) + labels->offset;
  p.loss = reinterpret_cast<float *>(const_cast<char *>(data_of(loss))) + loss->offset;
  p.softmax = softmax ? reinterpret_cast<float *>(const_cast<char *>(data_of(softmax))) + softmax->offset : nullptr;
  p.grad = grad ? reinterpret_cast<float *>(const_cast<char *>(data_of(grad))) + grad->offset : nullptr;
  p.rows = R;
  p.C = C;
  p.sx = logits->strides[0];
  p.ssm = softmax ? softmax->strides[0] : 0;
  p.sg = grad ? grad->strides[0] : 0;
  return noalloc ? launch_sce_noalloc(p, current_stream()) : launch_sce(p, current_stream());
}

template <typename D>
float *out_f32(D *d) {
  return reinterpret_cast<float *>(const_cast<char *>(data_of(d))) + d->offset;
}
template <typename D>
const float *in_f32(const D *d) {
  return reinterpret_cast<const float *>(data_of(d)) + d->offset;
}

}  // namespace

// Two operands are apart where their ranges are, or, views of one buffer, where
// modulo a step common to their longer strides what is left of each (the shorter
// strides and the runs) lies beside the other's.
static bool apart(const Extent &a, const Extent &b) {
  auto span = [](const Extent &x, int64_t below) {
    int64_t s = x.run;
    for (int i = 0; i < 3; ++i)
      if (x.n[i] > 1 && x.st[i] < below) s += (x.n[i] - 1) * x.st[i];
    return s;
  };
  if (!a.run || !b.run) return true;
  const intptr_t pa = reinterpret_cast<intptr_t>(a.p), pb = reinterpret_cast<intptr_t>(b.p);
  if (pa >= pb + span(b, INT64_MAX) || pb >= pa + span(a, INT64_MAX)) return true;
  for (const Extent *x : {&a, &b})
    for (int i = 0; i < 3; ++i) {
      const int64_t least = x->st[i];
      if (x->n[i] <= 1 || least == 0) continue;
      int64_t step = 0;
      for (const Extent *y : {&a, &b})
        for (int j = 0; j < 3; ++j)
          if (y->n[j] > 1 && y->st[j] >= least) step = std::gcd(step, y->st[j]);
      const int64_t at = ((pb - pa) % step + step) % step;
      if (at >= span(a, least) && step - at >= span(b, least)) return true;
    }
  return false;
}

int32_t check_apart(const char *w, const Extent &result,
                              std::initializer_list<Extent> others) {
  for (const Extent &x : others)
    if (!apart(result, x)) return fail(NOVA_HIP_EINVAL, "%s: %s overlaps %s", w, result.name, x.name);
  return NOVA_HIP_SUCCESS;
}
}  // namespace nova_hip

using namespace nova_hip;

extern "C" {

int32_t _mlir_ciface_nova_hip_gemm(const NovaMemRef3D *A, const NovaMemRef3D *B,
                                   NovaMemRef3D *C, const NovaMemRef1D *bias,
                                   int32_t flags) {
  return gemm_core(A, B, C, bias, flags);
}

int32_t _mlir_ciface_nova_hip_matmul_f32(const NovaMemRef2D *A, const NovaMemRef2D *B,
                                         NovaMemRef2D *C) {
  return gemm2d(A, B, C, nullptr,
                NOVA_HIP_GEMM_FLAGS(NOVA_HIP_DT_F32, NOVA_HIP_DT_F32, NOVA_HIP_EPI_NONE, 0));
}

int32_t _mlir_ciface_nova_hip_batch_matmul_f32(const NovaMemRef3D *A, const NovaMemRef3D *B,
                                               NovaMemRef3D *C) {
  return gemm_core(A, B, C, nullptr,
                   NOVA_HIP_GEMM_FLAGS(NOVA_HIP_DT_F32, NOVA_HIP_DT_F32, NOVA_HIP_EPI_NONE, 0));
}

int32_t _mlir_ciface_nova_hip_batch_matmul_bf16_f32(const NovaMemRef3D *A,
                                                    const NovaMemRef3D *B,
                                                    NovaMemRef3D *C) {
  return gemm_core(A, B, C, nullptr,
                   NOVA_HIP_GEMM_FLAGS(NOVA_HIP_DT_BF16, NOVA_HIP_DT_F32, NOVA_HIP_EPI_NONE, 0));
}

int32_t _mlir_ciface_nova_hip_batch_matmul_f16_f32(const NovaMemRef3D *A,
                                                   const NovaMemRef3D *B,
                                                   NovaMemRef3D *C) {
  return gemm_core(A, B, C, nullptr,
                   NOVA_HIP_GEMM_FLAGS(NOVA_HIP_DT_F16, NOVA_HIP_DT_F32, NOVA_HIP_EPI_NONE, 0));
}

int32_t _mlir_ciface_nova_hip_matmul_bf16_f32(const NovaMemRef2D *A, const NovaMemRef2D *B,
                                              NovaMemRef2D *C) {
  return gemm2d(A, B, C, nullptr,
                NOVA_HIP_GEMM_FLAGS(NOVA_HIP_DT_BF16, NOVA_HIP_DT_F32, NOVA_HIP_EPI_NONE, 0));
}

int32_t _mlir_ciface_nova_hip_matmul_f16_f32(const NovaMemRef2D *A, const NovaMemRef2D *B,
                                             NovaMemRef2D *C) {
  return gemm2d(A, B, C, nullptr,
                NOVA_HIP_GEMM_FLAGS(NOVA_HIP_DT_F16, NOVA_HIP_DT_F32, NOVA_HIP_EPI_NONE, 0));
}

int32_t _mlir_ciface_nova_hip_linear(const NovaMemRef2D *x, const NovaMemRef2D *weight,
                                     const NovaMemRef1D *bias, NovaMemRef2D *y,
                                     int32_t flags) {
  return gemm2d(x, weight, y, bias, flags);
}

int32_t _mlir_ciface_nova_hip_linear_bf16_bias_gelu(const NovaMemRef2D *x,
                                                    const NovaMemRef2D *weight,
                                                    const NovaMemRef1D *bias,
                                                    NovaMemRef2D *y) {
  return gemm2d(x, weight, y, bias,
                NOVA_HIP_GEMM_FLAGS(NOVA_HIP_DT_BF16, NOVA_HIP_DT_BF16,
                                    NOVA_HIP_EPI_BIAS_GELU, NOVA_HIP_DT_BF16));
}

int32_t _mlir_ciface_nova_hip_layer_norm_f32(const NovaMemRef2D *x, const NovaMemRef1D *gamma,
                                             const NovaMemRef1D *beta, NovaMemRef2D *y,
                                             NovaMemRef1D *mean_sum, NovaMemRef1D *rstd,
                                             float eps) {
  clear_error();
  if (!x || !gamma || !beta || !y) return fail(NOVA_HIP_EINVAL, "layer_norm: null descriptor");
  const int64_t R = x->sizes[0], D = x->sizes[1];
  if (R < 0 || D < 0) return fail(NOVA_HIP_ESHAPE, "layer_norm: negative size");
  if (y->sizes[0] != R || y->sizes[1] != D)
    return fail(NOVA_HIP_ESHAPE, "layer_norm: y shape differs from x");
  if (gamma->sizes[0] != D || beta->sizes[0] != D)
    return fail(NOVA_HIP_ESHAPE, "layer_norm: gamma/beta size != D");
  if (mean_sum && mean_sum->sizes[0] != R) return fail(NOVA_HIP_ESHAPE, "layer_norm: mean_sum size != rows");
  if (rstd && rstd->sizes[0] != R) return fail(NOVA_HIP_ESHAPE, "layer_norm: rstd size != rows");
  if (R == 0) return NOVA_HIP_SUCCESS;
  if (D == 0) return fail(NOVA_HIP_ESHAPE, "layer_norm: empty normalised dim");
  if ((x->strides[1] != 1 && D > 1) || (y->strides[1] != 1 && D > 1) ||
      (gamma->strides[0] != 1 && D > 1) || (beta->strides[0] != 1 && D > 1))
    return fail(NOVA_HIP_ESTRIDE, "layer_norm: last dim must be contiguous");
  if ((mean_sum && mean_sum->strides[0] != 1 && R > 1) || (rstd && rstd->strides[0] != 1 && R > 1))
    return fail(NOVA_HIP_ESTRIDE, "layer_norm: stats must be contiguous");
  if (!x->aligned || !y->aligned || !gamma->aligned || !beta->aligned ||
      (mean_sum && !mean_sum->aligned) || (rstd && !rstd->aligned))
    return fail(NOVA_HIP_EINVAL, "layer_norm: null data pointer");
  if ((R > 1 && (x->strides[0] < D || y->strides[0] < D)))
    return fail(NOVA_HIP_ESTRIDE, "layer_norm: rows overlap");
  LayerNormProblem p;
  p.x = reinterpret_cast<const float *>(data_of(x)) + x->offset;
  p.y = reinterpret_cast<float *>(const_cast<char *>(data_of(y))) + y->offset;
  p.gamma = reinterpret_cast<const float *>(data_of(gamma)) + gamma->offset;
  p.beta = reinterpret_cast<const float *>(data_of(beta)) + beta->offset;
  p.mean_sum = mean_sum ? reinterpret_cast<float *>(const_cast<char *>(data_of(mean_sum))) + mean_sum->offset : nullptr;
  p.rstd = rstd ? reinterpret_cast<float *>(const_cast<char *>(data_of(rstd))) + rstd->offset : nullptr;
  p.rows = R;
  p.D = D;
  p.sx = x->strides[0];
  p.sy = y->strides[0];
  p.eps = eps;
  return launch_layer_norm(p, current_stream());
}

int32_t _mlir_ciface_nova_hip_sce_f32(const NovaMemRef2D *logits, const NovaMemRef1D *labels,
                                      NovaMemRef1D *loss, NovaMemRef2D *softmax) {
  return sce_common(logits, labels, loss, softmax, nullptr, "sce");
}

int32_t _mlir_ciface_nova_hip_sce_f32_noalloc(const NovaMemRef2D *logits,
                                              const NovaMemRef1D *labels, NovaMemRef1D *loss,
                                              NovaMemRef2D *softmax) {
  return sce_common(logits, labels, loss, softmax, nullptr, "sce_noalloc", true);
}

int32_t _mlir_ciface_nova_hip_sce_fwd_bwd_f32(const NovaMemRef2D *logits,
                                              const NovaMemRef1D *labels, NovaMemRef1D *loss,
                                              NovaMemRef2D *grad) {
  if (!grad) {
    clear_error();
    return fail(NOVA_HIP_EINVAL, "sce_fwd_bwd: null grad descriptor");
  }
  return sce_common(logits, labels, loss, nullptr, grad, "sce_fwd_bwd");
}

int32_t _mlir_ciface_nova_hip_sce_backward_f32(const NovaMemRef2D *softmax,
                                               const NovaMemRef1D *labels, NovaMemRef2D *grad) {
  clear_error();
  if (!softmax || !labels || !grad) return fail(NOVA_HIP_EINVAL, "sce_backward: null descriptor");
  const int64_t R = softmax->sizes[0], C = softmax->sizes[1];
  if (R < 0 || C < 0) return fail(NOVA_HIP_ESHAPE, "sce_backward: negative size");
  if (labels->sizes[0] != R) return fail(NOVA_HIP_ESHAPE, "sce_backward: labels size != rows");
  if (grad->sizes[0] != R || grad->sizes[1] != C)
    return fail(NOVA_HIP_ESHAPE, "sce_backward: grad shape differs from softmax");
  if (R == 0 || C == 0) return NOVA_HIP_SUCCESS;
  if ((softmax->strides[1] != 1 && C > 1) || (grad->strides[1] != 1 && C > 1) ||
      (labels->strides[0] != 1 && R > 1))
    return fail(NOVA_HIP_ESTRIDE, "sce_backward: last dim must be contiguous");
  if (R > 1 && (softmax->strides[0] < C || grad->strides[0] < C))
    return fail(NOVA_HIP_ESTRIDE, "sce_backward: rows overlap");
  if (!softmax->aligned || !labels->aligned || !grad->aligned)
    return fail(NOVA_HIP_EINVAL, "sce_backward: null data pointer");
  SceBackwardProblem p;
  p.softmax = in_f32(softmax);
  p.labels = reinterpret_cast<const int32_t *>(data_of(labels)) + labels->offset;
  p.grad = out_f32(grad);
  p.rows = R;
  p.C = C;
  p.ss = softmax->strides[0];
  p.sg = grad->strides[0];
  return launch_sce_backward(p, current_stream());
}

int32_t _mlir_ciface_nova_hip_layer_norm_backward_f32(
    const NovaMemRef2D *grad_y, const NovaMemRef2D *x, const NovaMemRef1D *gamma,
    const NovaMemRef1D *mean_sum, const NovaMemRef1D *rstd, NovaMemRef2D *dx,
    NovaMemRef1D *dgamma, NovaMemRef1D *dbeta) {
  clear_error();
  const char *w = "layer_norm_backward";
  if (!grad_y || !x || !gamma || !mean_sum || !rstd)
    return fail(NOVA_HIP_EINVAL, "%s: null descriptor", w);
  const int64_t R = x->sizes[0], D = x->sizes[1];
  if (R < 0 || D < 0) return fail(NOVA_HIP_ESHAPE, "%s: negative size", w);
  if (grad_y->sizes[0] != R || grad_y->sizes[1] != D || (dx && (dx->sizes[0] != R || dx->sizes[1] != D)))
    return fail(NOVA_HIP_ESHAPE, "%s: grad_y / dx shape differs from x", w);
  if (gamma->sizes[0] != D || (dgamma && dgamma->sizes[0] != D) || (dbeta && dbeta->sizes[0] != D))
    return fail(NOVA_HIP_ESHAPE, "%s: gamma / dgamma / dbeta size != D", w);
  if (mean_sum->sizes[0] != R || rstd->sizes[0] != R)
    return fail(NOVA_HIP_ESHAPE, "%s: mean_sum / rstd size != rows", w);
  if (D == 0) return fail(NOVA_HIP_ESHAPE, "%s: empty normalised dim", w);
  if ((x->strides[1] != 1 && D > 1) || (grad_y->strides[1] != 1 && D > 1) ||
      (dx && dx->strides[1] != 1 && D > 1) || (gamma->strides[0] != 1 && D > 1) ||
      (dgamma && dgamma->strides[0] != 1 && D > 1) || (dbeta && dbeta->strides[0] != 1 && D > 1))
    return fail(NOVA_HIP_ESTRIDE, "%s: last dim must be contiguous", w);
  if ((mean_sum->strides[0] != 1 || rstd->strides[0] != 1) && R > 1)
    return fail(NOVA_HIP_ESTRIDE, "%s: stats must be contiguous", w);
  if (R > 1 && (x->strides[0] < D || grad_y->strides[0] < D || (dx && dx->strides[0] < D)))
    return fail(NOVA_HIP_ESTRIDE, "%s: rows overlap", w);
  if (!gamma->aligned || (dgamma && !dgamma->aligned) || (dbeta && !dbeta->aligned) ||
      (R > 0 && (!x->aligned || !grad_y->aligned || !mean_sum->aligned || !rstd->aligned ||
                 (dx && !dx->aligned))))
    return fail(NOVA_HIP_EINVAL, "%s: null data pointer", w);
  LayerNormBackwardProblem p;
  p.gy = in_f32(grad_y);
  p.x = in_f32(x);
  p.gamma = in_f32(gamma);
  p.mean_sum = in_f32(mean_sum);
  p.rstd = in_f32(rstd);
  p.dx = dx ? out_f32(dx) : nullptr;
  p.dgamma = dgamma ? out_f32(dgamma) : nullptr;
  p.dbeta = dbeta ? out_f32(dbeta) : nullptr;
  p.rows = R;
  p.D = D;
  p.sgy = grad_y->strides[0];
  p.sx = x->strides[0];
  p.sdx = dx ? dx->strides[0] : 0;
  return launch_layer_norm_backward(p, current_stream());
}

int32_t _mlir_ciface_nova_hip_linear_backward(const NovaMemRef2D *grad_out, const NovaMemRef2D *x,
                                              const NovaMemRef2D *weight,
                                              NovaMemRef2D *grad_input,
                                              NovaMemRef2D *grad_weight,
                                              NovaMemRef1D *grad_bias, int32_t flags) {
  clear_error();
  const char *w = "linear_backward";
  if (!grad_out || !x || !weight) return fail(NOVA_HIP_EINVAL, "%s: null descriptor", w);
  int in_dt, out_dt;
  int32_t rc = backward_flags(flags, in_dt, out_dt, w);
  if (rc) return rc;
  const int64_t M = x->sizes[0], K = x->sizes[1], N = weight->sizes[1];
  if (weight->sizes[0] != K || grad_out->sizes[0] != M || grad_out->sizes[1] != N)
    return fail(NOVA_HIP_ESHAPE, "%s: x [%lld,%lld], weight [%lld,%lld], grad_out [%lld,%lld]",
                w, (long long)M, (long long)K, (long long)weight->sizes[0], (long long)N,
                (long long)grad_out->sizes[0], (long long)grad_out->sizes[1]);
  // grad_input [M,K] = grad_out . weight^T  (NovaToLinalgGeneric.cpp:1867-1911)
  // grad_weight [K,N] = x^T . grad_out  (:1913-1968)
  // grad_bias [N] = column sums of grad_out  (:1970-1989)
  // Every requested output is validated before the first launch, so a call
  // that fails writes nothing.
  NovaMemRef2D wt = transposed(weight), xt = transposed(x);
  if (grad_input && (rc = gemm2d_to(grad_out, &wt, grad_input, flags, false))) return rc;
  if (grad_weight && (rc = gemm2d_to(&xt, grad_out, grad_weight, flags, false))) return rc;
  if (grad_bias) {
    clear_error();
    if (grad_bias->sizes[0] != N) return fail(NOVA_HIP_ESHAPE, "%s: grad_bias size != N", w);
    if (grad_bias->strides[0] != 1 && N > 1)
      return fail(NOVA_HIP_ESTRIDE, "%s: grad_bias must be contiguous", w);
    if (grad_out->strides[1] != 1 && N > 1)
      return fail(NOVA_HIP_ESTRIDE, "%s: grad_out must have unit stride on N for grad_bias", w);
    if (M > 1 && grad_out->strides[0] < N) return fail(NOVA_HIP_ESTRIDE, "%s: grad_out rows overlap", w);
    if (N > 0 && (!grad_bias->aligned || (M > 0 && !grad_out->aligned)))
      return fail(NOVA_HIP_EINVAL, "%s: null data pointer", w);
    if (!col_sum_in_range(M, N))
      return fail(NOVA_HIP_ERANGE, "%s: grad_bias of [%lld, %lld] exceeds the column sum's range",
                  w, (long long)M, (long long)N);
  }
  if (grad_input && (rc = gemm2d_to(grad_out, &wt, grad_input, flags))) return rc;
  if (grad_weight && (rc = gemm2d_to(&xt, grad_out, grad_weight, flags))) return rc;
  if (grad_bias) {
    ColSumProblem p;
    p.in = data_of(grad_out) + grad_out->offset * dtype_size(in_dt);
    p.out = const_cast<char *>(data_of(grad_bias)) + grad_bias->offset * dtype_size(out_dt);
    p.rows = M;
    p.cols = N;
    p.ld = grad_out->strides[0];
    p.in_dt = in_dt;
    p.out_dt = out_dt;
    if ((rc = launch_col_sum(p, current_stream()))) return rc;
  }
  return NOVA_HIP_SUCCESS;
}

int32_t _mlir_ciface_nova_hip_matmul_backward(const NovaMemRef2D *grad, const NovaMemRef2D *A,
                                              const NovaMemRef2D *B, NovaMemRef2D *grad_a,
                                              NovaMemRef2D *grad_b, int32_t flags) {
  clear_error();
  const char *w = "matmul_backward";
  if (!grad || !A || !B) return fail(NOVA_HIP_EINVAL, "%s: null descriptor", w);
  int in_dt, out_dt;
  int32_t rc = backward_flags(flags, in_dt, out_dt, w);
  if (rc) return rc;
  const int64_t M = A->sizes[0], K = A->sizes[1], N = B->sizes[1];
  if (B->sizes[0] != K || grad->sizes[0] != M || grad->sizes[1] != N)
    return fail(NOVA_HIP_ESHAPE, "%s: A [%lld,%lld], B [%lld,%lld], grad [%lld,%lld]", w,
                (long long)M, (long long)K, (long long)B->sizes[0], (long long)N,
                (long long)grad->sizes[0], (long long)grad->sizes[1]);
  // grad_a [M,K] = grad . B^T; grad_b [K,N] = A^T . grad
  // (NovaMatmulBackwardPattern, NovaToLinalgGeneric.cpp:160-239), both
  // validated before either is launched.
  NovaMemRef2D bt = transposed(B), at = transposed(A);
  if (grad_a && (rc = gemm2d_to(grad, &bt, grad_a, flags, false))) return rc;
  if (grad_b && (rc = gemm2d_to(&at, grad, grad_b, flags, false))) return rc;
  if (grad_a && (rc = gemm2d_to(grad, &bt, grad_a, flags))) return rc;
  if (grad_b && (rc = gemm2d_to(&at, grad, grad_b, flags))) return rc;
  return NOVA_HIP_SUCCESS;
}

// ---- program glue ---------------------------------------------------------------
namespace {
bool index_dt_ok(int32_t dt) {
  return dt == NOVA_HIP_DT_I16 || dt == NOVA_HIP_DT_I32 || dt == NOVA_HIP_DT_I64;
}
int index_size(int32_t dt) { return dt == NOVA_HIP_DT_I16 ? 2 : dt == NOVA_HIP_DT_I32 ? 4 : 8; }
// A dense 1-D f32 view (unit stride, or a single element).
int32_t dense1(const NovaMemRef1D *d, const char *w, const char *what) {
  if (!d) return fail(NOVA_HIP_EINVAL, "%s: null %s", w, what);
  if (d->sizes[0] < 0) return fail(NOVA_HIP_ESHAPE, "%s: negative size", w);
  if (d->sizes[0] > 1 && d->strides[0] != 1)
    return fail(NOVA_HIP_ESTRIDE, "%s: %s must be dense", w, what);
  if (d->sizes[0] > 0 && !d->aligned) return fail(NOVA_HIP_EINVAL, "%s: null data pointer", w);
  return NOVA_HIP_SUCCESS;
}
}  // namespace

int32_t _mlir_ciface_nova_hip_binary_f32(const NovaMemRef4D *a, const NovaMemRef4D *b,
                                         NovaMemRef4D *c, int32_t op) {
  clear_error();
  const char *w = "binary";
  if (!a || !b || !c) return fail(NOVA_HIP_EINVAL, "%s: null descriptor", w);
  if (op < NOVA_HIP_BIN_ADD || op > NOVA_HIP_BIN_DIV)
    return fail(NOVA_HIP_EINVAL, "%s: unknown op %d", w, op);
  BinaryProblem p;
  int64_t n = 1;
  for (int d = 0; d < 4; ++d) {
    const int64_t m = c->sizes[d];
    if (m < 0 || a->sizes[d] < 0 || b->sizes[d] < 0)
      return fail(NOVA_HIP_ESHAPE, "%s: negative size", w);
    if ((a->sizes[d] != m && a->sizes[d] != 1) || (b->sizes[d] != m && b->sizes[d] != 1))
      return fail(NOVA_HIP_ESHAPE, "%s: dim %d: %lld and %lld do not broadcast to %lld", w, d,
                  (long long)a->sizes[d], (long long)b->sizes[d], (long long)m);
    p.size[d] = m;
    p.sa[d] = a->sizes[d] == 1 ? 0 : a->strides[d];
    p.sb[d] = b->sizes[d] == 1 ? 0 : b->strides[d];
    p.sc[d] = c->strides[d];
    n *= m;
  }
  if (n == 0) return NOVA_HIP_SUCCESS;
  if (!a->aligned || !b->aligned || !c->aligned)
    return fail(NOVA_HIP_EINVAL, "%s: null data pointer", w);
  p.a = in_f32(a);
  p.b = in_f32(b);
  p.c = out_f32(c);
  p.op = op;
  return launch_binary(p, current_stream());
}

int32_t _mlir_ciface_nova_hip_fill_f32(NovaMemRef1D *out, float value) {
  clear_error();
  if (!out) return fail(NOVA_HIP_EINVAL, "fill: null descriptor");
  if (out->sizes[0] < 0) return fail(NOVA_HIP_ESHAPE, "fill: negative size");
  if (out->sizes[0] == 0) return NOVA_HIP_SUCCESS;
  if (!out->aligned) return fail(NOVA_HIP_EINVAL, "fill: null data pointer");
  return launch_fill(out_f32(out), out->sizes[0], out->strides[0], value, current_stream());
}

int32_t _mlir_ciface_nova_hip_gelu_f32(const NovaMemRef1D *x, NovaMemRef1D *y) {
  clear_error();
  int32_t rc;
  if ((rc = dense1(x, "gelu", "x")) || (rc = dense1(y, "gelu", "y"))) return rc;
  if (x->sizes[0] != y->sizes[0]) return fail(NOVA_HIP_ESHAPE, "gelu: sizes differ");
  return launch_gelu(in_f32(x), out_f32(y), x->sizes[0], current_stream());
}

int32_t _mlir_ciface_nova_hip_gelu_backward_f32(const NovaMemRef1D *grad_out,
                                                const NovaMemRef1D *x, NovaMemRef1D *out) {
  clear_error();
  const char *w = "gelu_backward";
  int32_t rc;
  if ((rc = dense1(grad_out, w, "grad_out")) || (rc = dense1(x, w, "x")) ||
      (rc = dense1(out, w, "out")))
    return rc;
  if (x->sizes[0] != grad_out->sizes[0] || x->sizes[0] != out->sizes[0])
    return fail(NOVA_HIP_ESHAPE, "%s: sizes differ", w);
  return launch_gelu_backward(in_f32(grad_out), in_f32(x), out_f32(out), x->sizes[0],
                              current_stream());
}

int32_t _mlir_ciface_nova_hip_gather_f32(const NovaMemRef2D *table, const NovaMemRef1D *idx,
                                         NovaMemRef2D *out, int32_t idx_dt) {
  clear_error();
  const char *w = "gather";
  if (!table || !idx || !out) return fail(NOVA_HIP_EINVAL, "%s: null descriptor", w);
  if (!index_dt_ok(idx_dt)) return fail(NOVA_HIP_EDTYPE, "%s: index dtype %d", w, idx_dt);
  if (!nonneg_sizes(table, 2) || !nonneg_sizes(idx, 1) || !nonneg_sizes(out, 2))
    return fail(NOVA_HIP_ESHAPE, "%s: negative size", w);
  const int64_t n = idx->sizes[0], D = table->sizes[1];
  if (out->sizes[0] != n || out->sizes[1] != D)
    return fail(NOVA_HIP_ESHAPE, "%s: out is [%lld, %lld], want [%lld, %lld]", w,
                (long long)out->sizes[0], (long long)out->sizes[1], (long long)n, (long long)D);
  if (n == 0 || D == 0) return NOVA_HIP_SUCCESS;
  if ((D > 1 && (table->strides[1] != 1 || out->strides[1] != 1)))
    return fail(NOVA_HIP_ESTRIDE, "%s: rows must be contiguous", w);
  if (!table->aligned || !idx->aligned || !out->aligned)
    return fail(NOVA_HIP_EINVAL, "%s: null data pointer", w);
  GatherProblem p;
  p.table = in_f32(table);
  p.idx = data_of(idx) + idx->offset * index_size(idx_dt);
  p.out = out_f32(out);
  p.rows = table->sizes[0];
  p.D = D;
  p.n = n;
  p.st = table->strides[0];
  p.so = out->strides[0];
  p.sidx = idx->strides[0];
  p.idx_dt = idx_dt;
  return launch_gather(p, current_stream());
}

int32_t _mlir_ciface_nova_hip_scatter_add_f32(NovaMemRef2D *out, const NovaMemRef1D *idx,
                                              const NovaMemRef2D *src, int32_t idx_dt) {
  clear_error();
  const char *w = "scatter_add";
  if (!out || !idx || !src) return fail(NOVA_HIP_EINVAL, "%s: null descriptor", w);
  if (!index_dt_ok(idx_dt)) return fail(NOVA_HIP_EDTYPE, "%s: index dtype %d", w, idx_dt);
  if (!nonneg_sizes(out, 2) || !nonneg_sizes(idx, 1) || !nonneg_sizes(src, 2))
    return fail(NOVA_HIP_ESHAPE, "%s: negative size", w);
  const int64_t n = idx->sizes[0], D = out->sizes[1];
  if (src->sizes[0] != n || src->sizes[1] != D)
    return fail(NOVA_HIP_ESHAPE, "%s: src is [%lld, %lld], want [%lld, %lld]", w,
                (long long)src->sizes[0], (long long)src->sizes[1], (long long)n, (long long)D);
  if (n == 0 || D == 0) return NOVA_HIP_SUCCESS;
  if (D > 1 && (out->strides[1] != 1 || src->strides[1] != 1))
    return fail(NOVA_HIP_ESTRIDE, "%s: rows must be contiguous", w);
  if (!out->aligned || !idx->aligned || !src->aligned)
    return fail(NOVA_HIP_EINVAL, "%s: null data pointer", w);
  ScatterAddProblem p;
  p.out = out_f32(out);
  p.idx = data_of(idx) + idx->offset * index_size(idx_dt);
  p.src = in_f32(src);
  p.rows = out->sizes[0];
  p.D = D;
  p.n = n;
  p.so = out->strides[0];
  p.ss = src->strides[0];
  p.sidx = idx->strides[0];
  p.idx_dt = idx_dt;
  return launch_scatter_add(p, current_stream());
}

int32_t _mlir_ciface_nova_hip_reduce_sum_f32(const NovaMemRef3D *x, NovaMemRef2D *out) {
  clear_error();
  const char *w = "reduce_sum";
  if (!x || !out) return fail(NOVA_HIP_EINVAL, "%s: null descriptor", w);
  if (!nonneg_sizes(x, 3) || !nonneg_sizes(out, 2))
    return fail(NOVA_HIP_ESHAPE, "%s: negative size", w);
  if (out->sizes[0] != x->sizes[0] || out->sizes[1] != x->sizes[2])
    return fail(NOVA_HIP_ESHAPE, "%s: out is [%lld, %lld], want [%lld, %lld]", w,
                (long long)out->sizes[0], (long long)out->sizes[1], (long long)x->sizes[0],
                (long long)x->sizes[2]);
  if (x->sizes[0] * x->sizes[2] == 0) return NOVA_HIP_SUCCESS;
  if (!x->aligned || !out->aligned) return fail(NOVA_HIP_EINVAL, "%s: null data pointer", w);
  ReduceSumProblem p;
  p.x = in_f32(x);
  p.out = out_f32(out);
  p.outer = x->sizes[0];
  p.n = x->sizes[1];
  p.inner = x->sizes[2];
  p.so = x->strides[0];
  p.sn = x->strides[1];
  p.si = x->strides[2];
  p.soo = out->strides[0];
  p.soi = out->strides[1];
  return launch_reduce_sum(p, current_stream());
}

int32_t _mlir_ciface_nova_hip_index_to_i32(const NovaMemRef1D *src, NovaMemRef1D *dst,
                                           int32_t src_dt) {
  clear_error();
  const char *w = "index_to_i32";
  if (!src || !dst) return fail(NOVA_HIP_EINVAL, "%s: null descriptor", w);
  if (!index_dt_ok(src_dt)) return fail(NOVA_HIP_EDTYPE, "%s: index dtype %d", w, src_dt);
  int32_t rc;
  if ((rc = dense1(dst, w, "dst"))) return rc;
  if (src->sizes[0] != dst->sizes[0]) return fail(NOVA_HIP_ESHAPE, "%s: sizes differ", w);
  if (src->sizes[0] == 0) return NOVA_HIP_SUCCESS;
  if (!src->aligned) return fail(NOVA_HIP_EINVAL, "%s: null data pointer", w);
  return launch_index_to_i32(data_of(src) + src->offset * index_size(src_dt), src->strides[0],
                             src_dt,
                             reinterpret_cast<int32_t *>(const_cast<char *>(data_of(dst))) +
                                 dst->offset,
                             src->sizes[0], current_stream());
}

// ---- attention --------------------------------------------------------------------
namespace {
constexpr int64_t kAttnMaxStride = 1 << 23;  // elements; 128 rows stay below 2^31 bytes

// One operand [T, heads, D]: unit stride on D, rows of whole 16-byte chunks at
// 16-byte aligned addresses.  A dim of extent 1 may have any stride: it gets
// the row's own length, so that the rows a tile holds behind the last one lie
// outside the operand, where loads return zero.
int32_t attn_operand(const NovaMemRef3D *d, const char *w, const char *what, bool out,
                     AttentionOperand &o) {
  if (!d) return fail(NOVA_HIP_EINVAL, "%s: null %s descriptor", w, what);
  if (!nonneg_sizes(d, 3)) return fail(NOVA_HIP_ESHAPE, "%s: negative size", w);
  const int64_t T = d->sizes[0], H = d->sizes[1], D = d->sizes[2];
  o.st = T > 1 ? d->strides[0] : (D + 7) / 8 * 8;
  o.sh = H > 1 ? d->strides[1] : 0;
  if (T > 0x7fffffff - (1 << 20) || H > 0xffff)
    return fail(NOVA_HIP_ERANGE, "%s: %s has more than 2^31 - 2^20 tokens or 65535 heads", w, what);
  if (T == 0 || H == 0 || D == 0) {
    o.p = nullptr;
    return NOVA_HIP_SUCCESS;
  }
  if (!d->aligned) return fail(NOVA_HIP_EINVAL, "%s: null %s data pointer", w, what);
  if (D > 1 && d->strides[2] != 1)
    return fail(NOVA_HIP_ESTRIDE, "%s: %s must have unit stride on the head dim", w, what);
  if ((T > 1 && o.st < D) || o.sh < 0)
    return fail(NOVA_HIP_ESTRIDE, "%s: rows of %s overlap", w, what);
  o.p = const_cast<char *>(data_of(d)) + d->offset * 2;
  if (o.st % 8 || o.sh % 8 || (reinterpret_cast<uintptr_t>(o.p) & 15u))
    return fail(NOVA_HIP_ESTRIDE, "%s: rows of %s must start at 16-byte aligned addresses", w, what);
  if (o.st > kAttnMaxStride)
    return fail(NOVA_HIP_ERANGE, "%s: token stride of %s exceeds 2^23 elements", w, what);
  if (out && H > 1) {
    const bool apart = o.sh >= D && (T <= 1 || (o.st <= o.sh ? o.sh >= (T - 1) * o.st + D
                                                             : o.st >= (H - 1) * o.sh + D));
    if (!apart) return fail(NOVA_HIP_ESTRIDE, "%s: rows of %s overlap", w, what);
  }
  return NOVA_HIP_SUCCESS;
}

bool dense_i32(const NovaMemRef1D *d) { return d->sizes[0] <= 1 || d->strides[0] == 1; }

// The checks attention and its backward share: q, k, v, offsets and lse.
int32_t attn_common(const NovaMemRef3D *q, const NovaMemRef3D *k, const NovaMemRef3D *v,
                    const NovaMemRef1D *q_off, const NovaMemRef1D *k_off, const NovaMemRef2D *lse,
                    float scale, int32_t causal, int32_t dt, const char *w, AttentionProblem &p) {
  int32_t rc;
  if (!q_off || !k_off) return fail(NOVA_HIP_EINVAL, "%s: null offsets descriptor", w);
  if (dt != NOVA_HIP_DT_BF16 && dt != NOVA_HIP_DT_F16)
    return fail(NOVA_HIP_EDTYPE, "%s: dtype %d (bf16 and f16 are provided)", w, dt);
  if (!(scale > 0.0f) || !(scale < INFINITY))
    return fail(NOVA_HIP_EINVAL, "%s: scale must be positive and finite", w);
  if (causal != 0 && causal != 1) return fail(NOVA_HIP_EINVAL, "%s: causal is %d", w, causal);
  if ((rc = attn_operand(q, w, "q", false, p.q)) || (rc = attn_operand(k, w, "k", false, p.k)) ||
      (rc = attn_operand(v, w, "v", false, p.v)))
    return rc;
  p.Tq = q->sizes[0];
  p.heads = q->sizes[1];
  p.D = q->sizes[2];
  p.Tk = k->sizes[0];
  p.kv_heads = k->sizes[1];
  if (k->sizes[2] != p.D || v->sizes[0] != p.Tk || v->sizes[1] != p.kv_heads || v->sizes[2] != p.D)
    return fail(NOVA_HIP_ESHAPE, "%s: q [%lld,%lld,%lld], k [%lld,%lld,%lld], v [%lld,%lld,%lld]", w,
                (long long)p.Tq, (long long)p.heads, (long long)p.D, (long long)p.Tk,
                (long long)p.kv_heads, (long long)k->sizes[2], (long long)v->sizes[0],
                (long long)v->sizes[1], (long long)v->sizes[2]);
  if (p.heads > 0 && (p.kv_heads == 0 || p.heads % p.kv_heads))
    return fail(NOVA_HIP_ESHAPE, "%s: %lld query heads do not share %lld key heads evenly", w,
                (long long)p.heads, (long long)p.kv_heads);
  if (p.D % 8 || p.D > 128)
    return fail(NOVA_HIP_ERANGE, "%s: head dim %lld is not a multiple of 8 up to 128", w,
                (long long)p.D);
  if (q_off->sizes[0] < 1 || q_off->sizes[0] != k_off->sizes[0])
    return fail(NOVA_HIP_ESHAPE, "%s: offsets must both be [sequences + 1]", w);
  if (!dense_i32(q_off) || !dense_i32(k_off))
    return fail(NOVA_HIP_ESTRIDE, "%s: offsets must be dense", w);
  if (!q_off->aligned || !k_off->aligned) return fail(NOVA_HIP_EINVAL, "%s: null offsets pointer", w);
  p.B = q_off->sizes[0] - 1;
  if (p.B >= (1 << 24)) return fail(NOVA_HIP_ERANGE, "%s: more than 2^24 - 1 sequences", w);
  p.q_off = reinterpret_cast<const int32_t *>(data_of(q_off)) + q_off->offset;
  p.k_off = reinterpret_cast<const int32_t *>(data_of(k_off)) + k_off->offset;
  p.lse = nullptr;
  p.slse = 0;
  if (lse) {
    if (lse->sizes[0] != p.heads || lse->sizes[1] != p.Tq)
      return fail(NOVA_HIP_ESHAPE, "%s: lse must be [heads, query tokens]", w);
    if ((p.Tq > 1 && lse->strides[1] != 1) || (p.heads > 1 && lse->strides[0] < p.Tq))
      return fail(NOVA_HIP_ESTRIDE, "%s: lse rows must be dense and not overlap", w);
    if (!lse->aligned && p.heads * p.Tq > 0)
      return fail(NOVA_HIP_EINVAL, "%s: null lse pointer", w);
    p.lse = reinterpret_cast<float *>(const_cast<char *>(data_of(lse))) + lse->offset;
    p.slse = lse->strides[0];
  }
  p.scale = scale;
  p.causal = causal != 0;
  p.dt = dt;
  return NOVA_HIP_SUCCESS;
}

int32_t same_shape(const NovaMemRef3D *a, const NovaMemRef3D *b, const char *w, const char *what) {
  if (!a) return fail(NOVA_HIP_EINVAL, "%s: null %s descriptor", w, what);
  for (int i = 0; i < 3; ++i)
    if (a->sizes[i] != b->sizes[i]) return fail(NOVA_HIP_ESHAPE, "%s: shape of %s", w, what);
  return NOVA_HIP_SUCCESS;
}
}  // namespace

int32_t _mlir_ciface_nova_hip_attention(const NovaMemRef3D *q, const NovaMemRef3D *k,
                                        const NovaMemRef3D *v, const NovaMemRef1D *q_offsets,
                                        const NovaMemRef1D *k_offsets, NovaMemRef3D *out,
                                        NovaMemRef2D *lse, float scale, int32_t causal,
                                        int32_t dt) {
  clear_error();
  const char *w = "attention";
  AttentionProblem p;
  int32_t rc = attn_common(q, k, v, q_offsets, k_offsets, lse, scale, causal, dt, w, p);
  if (rc || (rc = same_shape(out, q, w, "out")) || (rc = attn_operand(out, w, "out", true, p.o)))
    return rc;
  return launch_attention(p, current_stream());
}

int64_t nova_hip_attention_backward_scratch(int64_t q_tokens, int64_t k_tokens, int64_t sequences,
                                            int64_t heads, int64_t kv_heads, int64_t D,
                                            int32_t causal) {
  if (q_tokens < 0 || k_tokens < 0 || sequences < 0 || heads <= 0 || kv_heads <= 0 || D <= 0 ||
      q_tokens > 0x7fffffff || k_tokens > 0x7fffffff || sequences > (1 << 24) || heads > 0xffff ||
      kv_heads > heads || D > 128)
    return 0;  // the call itself refuses these, or has nothing to do
  return attention_backward_scratch(q_tokens, k_tokens, sequences, heads, kv_heads, D, causal != 0);
}

int32_t _mlir_ciface_nova_hip_attention_backward(
    const NovaMemRef3D *grad_out, const NovaMemRef3D *q, const NovaMemRef3D *k,
    const NovaMemRef3D *v, const NovaMemRef3D *out, const NovaMemRef2D *lse,
    const NovaMemRef1D *q_offsets, const NovaMemRef1D *k_offsets, NovaMemRef3D *dq,
    NovaMemRef3D *dk, NovaMemRef3D *dv, NovaMemRef1D *scratch, float scale, int32_t causal,
    int32_t dt) {
  clear_error();
  const char *w = "attention_backward";
  if (!lse) return fail(NOVA_HIP_EINVAL, "%s: null lse descriptor", w);
  AttentionBackwardProblem p;
  int32_t rc = attn_common(q, k, v, q_offsets, k_offsets, lse, scale, causal, dt, w, p.f);
  if (rc || (rc = same_shape(out, q, w, "out")) || (rc = same_shape(grad_out, q, w, "grad_out")) ||
      (rc = same_shape(dq, q, w, "dq")) || (rc = same_shape(dk, k, w, "dk")) ||
      (rc = same_shape(dv, k, w, "dv")) || (rc = attn_operand(out, w, "out", false, p.f.o)) ||
      (rc = attn_operand(grad_out, w, "grad_out", false, p.go)) ||
      (rc = attn_operand(dq, w, "dq", true, p.dq)) || (rc = attn_operand(dk, w, "dk", true, p.dk)) ||
      (rc = attn_operand(dv, w, "dv", true, p.dv)))
    return rc;
  if (!scratch) return fail(NOVA_HIP_EINVAL, "%s: null scratch descriptor", w);
  if ((rc = dense1(scratch, w, "scratch"))) return rc;
  const int64_t need = nova_hip_attention_backward_scratch(p.f.Tq, p.f.Tk, p.f.B, p.f.heads,
                                                           p.f.kv_heads, p.f.D, causal);
  if (scratch->sizes[0] < need)
    return fail(NOVA_HIP_ESHAPE, "%s: scratch holds %lld floats, %lld are needed", w,
                (long long)scratch->sizes[0], (long long)need);
  p.scratch = out_f32(scratch);
  return launch_attention_backward(p, current_stream());
}

int64_t nova_hip_attention_decode_scratch(int64_t sequences, int64_t cache, int64_t heads,
                                          int64_t kv_heads, int64_t D) {
  if (sequences <= 0 || cache <= 0 || heads <= 0 || kv_heads <= 0 || D <= 0) return 0;
  if (sequences > 0xffff || cache > 0x7fffffff || heads > 0xffff || kv_heads > heads || D > 128)
    return 0;  // the call itself refuses these
  return attention_decode_scratch(sequences, cache, heads, kv_heads, D);
}

int32_t _mlir_ciface_nova_hip_attention_decode(const NovaMemRef3D *q, const NovaMemRef4D *k,
                                               const NovaMemRef4D *v, const NovaMemRef1D *lengths,
                                               NovaMemRef3D *out, NovaMemRef2D *lse,
                                               NovaMemRef1D *scratch, float scale, int32_t dt) {
  clear_error();
  const char *w = "attention_decode";
  if (!q || !k || !v || !lengths || !out) return fail(NOVA_HIP_EINVAL, "%s: null descriptor", w);
  if (dt != NOVA_HIP_DT_BF16 && dt != NOVA_HIP_DT_F16)
    return fail(NOVA_HIP_EDTYPE, "%s: dtype %d (bf16 and f16 are provided)", w, dt);
  if (!(scale > 0.0f) || !(scale < INFINITY))
    return fail(NOVA_HIP_EINVAL, "%s: scale must be positive and finite", w);
  if (!nonneg_sizes(q, 3) || !nonneg_sizes(k, 4) || !nonneg_sizes(v, 4) || !nonneg_sizes(out, 3) ||
      !nonneg_sizes(lengths, 1))
    return fail(NOVA_HIP_ESHAPE, "%s: negative size", w);
  AttentionDecodeProblem p;
  p.B = q->sizes[0];
  p.heads = q->sizes[1];
  p.D = q->sizes[2];
  p.S = k->sizes[1];
  p.kv_heads = k->sizes[2];
  for (int i = 0; i < 4; ++i)
    if (k->sizes[i] != v->sizes[i]) return fail(NOVA_HIP_ESHAPE, "%s: shapes of k and v differ", w);
  if (k->sizes[0] != p.B || k->sizes[3] != p.D || lengths->sizes[0] != p.B)
    return fail(NOVA_HIP_ESHAPE, "%s: q [%lld,%lld,%lld], k [%lld,%lld,%lld,%lld], lengths [%lld]", w,
                (long long)p.B, (long long)p.heads, (long long)p.D, (long long)k->sizes[0],
                (long long)p.S, (long long)p.kv_heads, (long long)k->sizes[3],
                (long long)lengths->sizes[0]);
  int32_t rc = same_shape(out, q, w, "out");
  if (rc) return rc;
  if (p.heads > 0 && (p.kv_heads == 0 || p.heads % p.kv_heads))
    return fail(NOVA_HIP_ESHAPE, "%s: %lld query heads do not share %lld key heads evenly", w,
                (long long)p.heads, (long long)p.kv_heads);
  if (p.D % 8 || p.D > 128)
    return fail(NOVA_HIP_ERANGE, "%s: head dim %lld is not a multiple of 8 up to 128", w,
                (long long)p.D);
  if (p.B > 0xffff || p.heads > 0xffff || p.S > 0x7fffffff - (1 << 20))
    return fail(NOVA_HIP_ERANGE, "%s: more than 65535 sequences or heads, or 2^31 - 2^20 rows", w);
  if (!dense_i32(lengths)) return fail(NOVA_HIP_ESTRIDE, "%s: lengths must be dense", w);
  if (lse && (lse->sizes[0] != p.B || lse->sizes[1] != p.heads))
    return fail(NOVA_HIP_ESHAPE, "%s: lse must be [sequences, heads]", w);
  if (p.B == 0 || p.heads == 0 || p.D == 0) return NOVA_HIP_SUCCESS;
  if (!q->aligned || !out->aligned || !lengths->aligned || (lse && !lse->aligned) ||
      (p.S > 0 && (!k->aligned || !v->aligned)))
    return fail(NOVA_HIP_EINVAL, "%s: null data pointer", w);
  // A dim of extent 1 may have any stride (see attn_operand).
  auto stride = [&](int64_t size, int64_t s) { return size > 1 ? s : p.D; };
  p.sqb = stride(p.B, q->strides[0]);
  p.sqh = stride(p.heads, q->strides[1]);
  p.sob = stride(p.B, out->strides[0]);
  p.soh = stride(p.heads, out->strides[1]);
  p.skb = stride(p.B, k->strides[0]);
  p.skt = stride(p.S, k->strides[1]);
  p.skh = stride(p.kv_heads, k->strides[2]);
  p.svb = stride(p.B, v->strides[0]);
  p.svt = stride(p.S, v->strides[1]);
  p.svh = stride(p.kv_heads, v->strides[2]);
  p.q = data_of(q) + q->offset * 2;
  p.k = data_of(k) + k->offset * 2;
  p.v = data_of(v) + v->offset * 2;
  p.o = const_cast<char *>(data_of(out)) + out->offset * 2;
  if (p.D > 1 && (q->strides[2] != 1 || out->strides[2] != 1 ||
                  (p.S > 0 && (k->strides[3] != 1 || v->strides[3] != 1))))
    return fail(NOVA_HIP_ESTRIDE, "%s: operands must have unit stride on the head dim", w);
  if (p.S == 0) {  // no rows to address
    p.k = p.v = nullptr;
    p.skb = p.skt = p.skh = p.svb = p.svt = p.svh = p.D;
  }
  if (p.sqb < 0 || p.skb < 0 || p.svb < 0 || p.skh < 0 || p.svh < 0 ||
      (p.heads > 1 && (p.sqh < p.D || p.soh < p.D)) ||
      (p.S > 1 && (p.skt < p.D || p.svt < p.D)))
    return fail(NOVA_HIP_ESTRIDE, "%s: rows overlap", w);
  if (p.B > 1 && p.sob < p.D) return fail(NOVA_HIP_ESTRIDE, "%s: rows of out overlap", w);
  if (p.B > 1 && p.heads > 1 &&
      (p.soh <= p.sob ? p.sob < (p.heads - 1) * p.soh + p.D : p.soh < (p.B - 1) * p.sob + p.D))
    return fail(NOVA_HIP_ESTRIDE, "%s: rows of out overlap", w);
  const int64_t any = p.sqb | p.sqh | p.sob | p.soh | p.skb | p.skt | p.skh | p.svb | p.svt | p.svh;
  if (any % 8 || ((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) |
                   reinterpret_cast<uintptr_t>(p.v) | reinterpret_cast<uintptr_t>(p.o)) & 15u))
    return fail(NOVA_HIP_ESTRIDE, "%s: rows must start at 16-byte aligned addresses", w);
  if (p.sqh > kAttnMaxStride || p.skt > kAttnMaxStride || p.svt > kAttnMaxStride)
    return fail(NOVA_HIP_ERANGE, "%s: a row stride exceeds 2^23 elements", w);
  p.lens = reinterpret_cast<const int32_t *>(data_of(lengths)) + lengths->offset;
  p.lse = nullptr;
  p.slse = 0;
  if (lse) {
    if ((p.heads > 1 && lse->strides[1] != 1) || (p.B > 1 && lse->strides[0] < p.heads))
      return fail(NOVA_HIP_ESTRIDE, "%s: lse rows must be dense and not overlap", w);
    p.lse = out_f32(lse);
    p.slse = lse->strides[0];
  }
  p.partial = nullptr;
  const int64_t need =
      nova_hip_attention_decode_scratch(p.B, p.S, p.heads, p.kv_heads, p.D);
  if (need > 0) {
    if (!scratch) return fail(NOVA_HIP_EINVAL, "%s: null scratch descriptor", w);
    if ((rc = dense1(scratch, w, "scratch"))) return rc;
    if (scratch->sizes[0] < need)
      return fail(NOVA_HIP_ESHAPE, "%s: scratch holds %lld floats, %lld are needed", w,
                  (long long)scratch->sizes[0], (long long)need);
    p.partial = out_f32(scratch);
    if (reinterpret_cast<uintptr_t>(p.partial) & 7u)
      return fail(NOVA_HIP_ESTRIDE, "%s: scratch must be 8-byte aligned", w);
  }
  p.scale = scale;
  p.dt = dt;
  return launch_attention_decode(p, current_stream());
}

// ---- losses over token log-probabilities ---------------------------------------------
namespace {
// logits [R, C], labels [R] and the optional gradient, shared by the three losses.
int32_t token_common(const NovaMemRef2D *logits, const NovaMemRef1D *labels, NovaMemRef2D *grad,
                     int32_t dt, const char *w, TokenLossProblem &p) {
  if (!logits || !labels) return fail(NOVA_HIP_EINVAL, "%s: null descriptor", w);
  if (dt != NOVA_HIP_DT_F32 && dt != NOVA_HIP_DT_BF16 && dt != NOVA_HIP_DT_F16)
    return fail(NOVA_HIP_EDTYPE, "%s: dtype %d (f32, bf16 and f16 are provided)", w, dt);
  p.rows = logits->sizes[0];
  p.C = logits->sizes[1];
  if (p.rows < 0 || p.C < 0) return fail(NOVA_HIP_ESHAPE, "%s: negative size", w);
  if (p.C == 0) return fail(NOVA_HIP_ESHAPE, "%s: zero classes", w);
  if (labels->sizes[0] != p.rows) return fail(NOVA_HIP_ESHAPE, "%s: labels size != rows", w);
  if (grad && (grad->sizes[0] != p.rows || grad->sizes[1] != p.C))
    return fail(NOVA_HIP_ESHAPE, "%s: grad shape differs from logits", w);
  if ((p.C > 1 && (logits->strides[1] != 1 || (grad && grad->strides[1] != 1))) ||
      (p.rows > 1 && labels->strides[0] != 1))
    return fail(NOVA_HIP_ESTRIDE, "%s: last dim must be contiguous", w);
  if (p.rows > 1 && (logits->strides[0] < p.C || (grad && grad->strides[0] < p.C)))
    return fail(NOVA_HIP_ESTRIDE, "%s: rows overlap", w);
  if (p.rows > 0 && (!logits->aligned || !labels->aligned || (grad && !grad->aligned)))
    return fail(NOVA_HIP_EINVAL, "%s: null data pointer", w);
  const int sz = dtype_size(dt);
  p.logits = data_of(logits) + logits->offset * sz;
  p.grad = grad ? const_cast<char *>(data_of(grad)) + grad->offset * sz : nullptr;
  p.labels = reinterpret_cast<const int32_t *>(data_of(labels)) + labels->offset;
  p.sx = logits->strides[0];
  p.sg = grad ? grad->strides[0] : 0;
  p.dt = dt;
  return NOVA_HIP_SUCCESS;
}

// The gradient apart from the logits, or column ranges of the same rows.
int32_t grad_apart(const TokenLossProblem &p, const char *w) {
  if (!p.grad || p.rows == 0) return NOVA_HIP_SUCCESS;
  const int64_t sz = dtype_size(p.dt), sx = p.rows > 1 ? p.sx : p.C, sg = p.rows > 1 ? p.sg : p.C;
  const intptr_t x = reinterpret_cast<intptr_t>(p.logits), g = reinterpret_cast<intptr_t>(p.grad);
  if (x >= g + ((p.rows - 1) * sg + p.C) * sz || g >= x + ((p.rows - 1) * sx + p.C) * sz)
    return NOVA_HIP_SUCCESS;
  const int64_t pitch = sx * sz, row = p.C * sz, at = ((g - x) % pitch + pitch) % pitch;
  if (sx == sg && at >= row && pitch - at >= row) return NOVA_HIP_SUCCESS;
  return fail(NOVA_HIP_EINVAL, "%s: grad overlaps logits", w);
}

// A dense f32 vector of n values.
int32_t vector_f32(const NovaMemRef1D *d, int64_t n, const char *w, const char *what) {
  int32_t rc = dense1(d, w, what);
  if (rc) return rc;
  if (d->sizes[0] != n)
    return fail(NOVA_HIP_ESHAPE, "%s: %s has %lld values, not %lld", w, what,
                (long long)d->sizes[0], (long long)n);
  return NOVA_HIP_SUCCESS;
}
}  // namespace

int32_t _mlir_ciface_nova_hip_token_logp(const NovaMemRef2D *logits, const NovaMemRef1D *labels,
                                         NovaMemRef1D *logp, NovaMemRef1D *lse, int32_t dt) {
  clear_error();
  const char *w = "token_logp";
  TokenLossProblem p;
  int32_t rc = token_common(logits, labels, nullptr, dt, w, p);
  if (rc || (rc = vector_f32(logp, p.rows, w, "logp")) ||
      (lse && (rc = vector_f32(lse, p.rows, w, "lse"))))
    return rc;
  return launch_token_logp(p, out_f32(logp), lse ? out_f32(lse) : nullptr, current_stream());
}

int32_t _mlir_ciface_nova_hip_policy_loss(
    const NovaMemRef2D *logits, const NovaMemRef1D *labels, const NovaMemRef1D *old_logp,
    const NovaMemRef1D *ref_logp, const NovaMemRef1D *advantage, const NovaMemRef1D *weight,
    NovaMemRef1D *loss, NovaMemRef1D *logp, NovaMemRef1D *row_loss, NovaMemRef2D *grad,
    float clip_low, float clip_high, float kl_coef, float grad_scale, int32_t dt) {
  clear_error();
  const char *w = "policy_loss";
  PolicyProblem p;
  int32_t rc = token_common(logits, labels, grad, dt, w, p.t);
  const int64_t R = p.t.rows;
  if (rc || (rc = vector_f32(old_logp, R, w, "old_logp")) ||
      (ref_logp && (rc = vector_f32(ref_logp, R, w, "ref_logp"))) ||
      (rc = vector_f32(advantage, R, w, "advantage")) || (rc = vector_f32(weight, R, w, "weight")) ||
      (rc = vector_f32(loss, 1, w, "loss")) || (rc = vector_f32(logp, R, w, "logp")) ||
      (rc = vector_f32(row_loss, R, w, "row_loss")))
    return rc;
  if (!(clip_low >= 0.0f && clip_low <= 1.0f) || !(clip_high >= 0.0f && clip_high < INFINITY))
    return fail(NOVA_HIP_EINVAL, "%s: clip_low must be in [0, 1], clip_high finite and >= 0", w);
  if (!std::isfinite(kl_coef) || !std::isfinite(grad_scale))
    return fail(NOVA_HIP_EINVAL, "%s: kl_coef and grad_scale must be finite", w);
  if (!ref_logp && kl_coef != 0.0f)
    return fail(NOVA_HIP_EINVAL, "%s: the KL term needs ref_logp", w);
  p.old_logp = in_f32(old_logp);
  p.ref_logp = ref_logp && kl_coef != 0.0f ? in_f32(ref_logp) : nullptr;
  p.advantage = in_f32(advantage);
  p.weight = in_f32(weight);
  p.loss = out_f32(loss);
  p.logp = out_f32(logp);
  p.row_loss = out_f32(row_loss);
  p.clip_low = clip_low;
  p.clip_high = clip_high;
  p.kl_coef = kl_coef;
  p.grad_scale = grad_scale;
  if ((rc = grad_apart(p.t, w))) return rc;
  return launch_policy_loss(p, current_stream());
}

int32_t _mlir_ciface_nova_hip_preference_loss(
    const NovaMemRef2D *logits, const NovaMemRef1D *labels, const NovaMemRef1D *offsets,
    const NovaMemRef1D *ref_logp, NovaMemRef1D *loss, NovaMemRef1D *seq_logp,
    NovaMemRef1D *pair_loss, NovaMemRef2D *token, NovaMemRef2D *grad, float beta, float smoothing,
    float grad_scale, int32_t dt) {
  clear_error();
  const char *w = "preference_loss";
  PreferenceProblem p;
  int32_t rc = token_common(logits, labels, grad, dt, w, p.t);
  if (rc) return rc;
  if (!offsets || !token) return fail(NOVA_HIP_EINVAL, "%s: null descriptor", w);
  const int64_t n = offsets->sizes[0] - 1;  // sequences
  if (n < 2 || n % 2)
    return fail(NOVA_HIP_ESHAPE, "%s: offsets must be [2 pairs + 1], at least one pair", w);
  p.pairs = n / 2;
  // A grid's dimension holds less than 2^32 threads, 256 to a pair.
  if (p.pairs >= (1 << 24)) return fail(NOVA_HIP_ERANGE, "%s: more than 2^24 - 1 pairs", w);
  if (!dense_i32(offsets)) return fail(NOVA_HIP_ESTRIDE, "%s: offsets must be dense", w);
  if (!offsets->aligned) return fail(NOVA_HIP_EINVAL, "%s: null offsets pointer", w);
  if ((rc = vector_f32(ref_logp, n, w, "ref_logp")) || (rc = vector_f32(loss, 1, w, "loss")) ||
      (rc = vector_f32(seq_logp, n, w, "seq_logp")) ||
      (rc = vector_f32(pair_loss, p.pairs, w, "pair_loss")))
    return rc;
  const int64_t R = p.t.rows;
  if (token->sizes[0] != 3 || token->sizes[1] != R)
    return fail(NOVA_HIP_ESHAPE, "%s: token must be [3, rows]", w);
  if ((R > 1 && token->strides[1] != 1) || token->strides[0] < R)
    return fail(NOVA_HIP_ESTRIDE, "%s: token rows must be dense and not overlap", w);
  if (R > 0 && !token->aligned) return fail(NOVA_HIP_EINVAL, "%s: null token pointer", w);
  if (!(beta > 0.0f && beta < INFINITY) || !(smoothing >= 0.0f && smoothing <= 1.0f) ||
      !std::isfinite(grad_scale))
    return fail(NOVA_HIP_EINVAL,
                "%s: beta must be positive, smoothing in [0, 1], grad_scale finite", w);
  p.offsets = reinterpret_cast<const int32_t *>(data_of(offsets)) + offsets->offset;
  p.ref_logp = in_f32(ref_logp);
  p.loss = out_f32(loss);
  p.seq_logp = out_f32(seq_logp);
  p.pair_loss = out_f32(pair_loss);
  p.logp = out_f32(token);
  p.lse = p.logp + token->strides[0];
  p.slope = p.lse + token->strides[0];
  p.beta = beta;
  p.smoothing = smoothing;
  p.grad_scale = grad_scale;
  if ((rc = grad_apart(p.t, w))) return rc;
  return launch_preference_loss(p, current_stream());
}

void nova_hip_set_stream(void *stream) { t_stream = static_cast<hipStream_t>(stream); }

void *nova_hip_get_stream(void) { return t_stream; }

int32_t nova_hip_synchronize(void) {
  clear_error();
  return check_hip(hipStreamSynchronize(t_stream), "synchronize");
}

const char *nova_hip_last_error(void) { return t_err; }

// ---- Typed aliases for lowered modules --------------------------------------
// A module declares each callee once, with one type; these aliases give the
// generic entry points one name per operand dtype combination.  The flags
// must name the alias's dtypes (the bias dtype only when the epilogue has a
// bias).
#define NOVA_GEMM_ALIAS(SUF, IN, OUT, BIAS)                                                    \
  int32_t _mlir_ciface_nova_hip_gemm_##SUF(const NovaMemRef3D *A, const NovaMemRef3D *B,       \
                                           NovaMemRef3D *C, const NovaMemRef1D *bias,          \
                                           int32_t flags) {                                    \
    const int epi = (flags >> 8) & 0xf;                                                        \
    const bool has_bias = epi == NOVA_HIP_EPI_BIAS || epi == NOVA_HIP_EPI_BIAS_GELU;          \
    if ((flags & 0xf) != (IN) || ((flags >> 4) & 0xf) != (OUT) ||                              \
        (has_bias && ((flags >> 12) & 0xf) != (BIAS))) {                                       \
      clear_error();                                                                           \
      return fail(NOVA_HIP_EINVAL, "gemm_" #SUF ": flags 0x%x name other dtypes", flags);     \
    }                                                                                          \
    return gemm_core(A, B, C, bias, flags);                                                    \
  }
#define NOVA_GEMM_ALIASES_OUT(IS, IN, OS, OUT)               \
  NOVA_GEMM_ALIAS(IS##_##OS##_bf32, IN, OUT, NOVA_HIP_DT_F32) \
  NOVA_GEMM_ALIAS(IS##_##OS##_bbf16, IN, OUT, NOVA_HIP_DT_BF16) \
  NOVA_GEMM_ALIAS(IS##_##OS##_bf16, IN, OUT, NOVA_HIP_DT_F16)
#define NOVA_GEMM_ALIASES_IN(IS, IN)                     \
  NOVA_GEMM_ALIASES_OUT(IS, IN, f32, NOVA_HIP_DT_F32)   \
  NOVA_GEMM_ALIASES_OUT(IS, IN, bf16, NOVA_HIP_DT_BF16) \
  NOVA_GEMM_ALIASES_OUT(IS, IN, f16, NOVA_HIP_DT_F16)
NOVA_GEMM_ALIASES_IN(f32, NOVA_HIP_DT_F32)
NOVA_GEMM_ALIASES_IN(bf16, NOVA_HIP_DT_BF16)
NOVA_GEMM_ALIASES_IN(f16, NOVA_HIP_DT_F16)

#define NOVA_BWD_ALIAS(SUF, IN, OUT)                                                             \
  int32_t _mlir_ciface_nova_hip_linear_backward_##SUF(                                           \
      const NovaMemRef2D *go, const NovaMemRef2D *x, const NovaMemRef2D *w, NovaMemRef2D *gi,    \
      NovaMemRef2D *gw, NovaMemRef1D *gb, int32_t flags) {                                       \
    if ((flags & 0xf) != (IN) || ((flags >> 4) & 0xf) != (OUT)) {                                \
      clear_error();                                                                             \
      return fail(NOVA_HIP_EINVAL, "linear_backward_" #SUF ": flags 0x%x name other dtypes",    \
                  flags);                                                                        \
    }                                                                                            \
    return _mlir_ciface_nova_hip_linear_backward(go, x, w, gi, gw, gb, flags);                  \
  }                                                                                              \
  int32_t _mlir_ciface_nova_hip_matmul_backward_##SUF(const NovaMemRef2D *g,                     \
                                                      const NovaMemRef2D *A,                     \
                                                      const NovaMemRef2D *B, NovaMemRef2D *ga,   \
                                                      NovaMemRef2D *gb, int32_t flags) {         \
    if ((flags & 0xf) != (IN) || ((flags >> 4) & 0xf) != (OUT)) {                                \
      clear_error();                                                                             \
      return fail(NOVA_HIP_EINVAL, "matmul_backward_" #SUF ": flags 0x%x name other dtypes",    \
                  flags);                                                                        \
    }                                                                                            \
    return _mlir_ciface_nova_hip_matmul_backward(g, A, B, ga, gb, flags);                       \
  }
NOVA_BWD_ALIAS(f32_f32, NOVA_HIP_DT_F32, NOVA_HIP_DT_F32)
NOVA_BWD_ALIAS(bf16_f32, NOVA_HIP_DT_BF16, NOVA_HIP_DT_F32)
NOVA_BWD_ALIAS(bf16_bf16, NOVA_HIP_DT_BF16, NOVA_HIP_DT_BF16)
NOVA_BWD_ALIAS(bf16_f16, NOVA_HIP_DT_BF16, NOVA_HIP_DT_F16)
NOVA_BWD_ALIAS(f16_f32, NOVA_HIP_DT_F16, NOVA_HIP_DT_F32)
NOVA_BWD_ALIAS(f16_bf16, NOVA_HIP_DT_F16, NOVA_HIP_DT_BF16)
NOVA_BWD_ALIAS(f16_f16, NOVA_HIP_DT_F16, NOVA_HIP_DT_F16)

int32_t _mlir_ciface_nova_hip_index_to_i32_i16(const NovaMemRef1D *src, NovaMemRef1D *dst,
                                               int32_t src_dt) {
  return _mlir_ciface_nova_hip_index_to_i32(src, dst, src_dt);
}
int32_t _mlir_ciface_nova_hip_index_to_i32_i64(const NovaMemRef1D *src, NovaMemRef1D *dst,
                                               int32_t src_dt) {
  return _mlir_ciface_nova_hip_index_to_i32(src, dst, src_dt);
}

int32_t _mlir_ciface_nova_hip_sce_loss_f32(const NovaMemRef2D *logits,
                                           const NovaMemRef1D *labels, NovaMemRef1D *loss) {
  return sce_common(logits, labels, loss, nullptr, nullptr, "sce");
}

const char *nova_hip_version(void) { return "libnova_hip 0.1.0 (gfx950)"; }

int32_t nova_hip_release_workspace(void) {
  clear_error();
  std::vector<hipStream_t> streams;
  {
    std::lock_guard<std::mutex> lock(g_ws_mu);
    for (auto &kv : g_ws) streams.push_back(kv.first);
  }
  int32_t rc = NOVA_HIP_SUCCESS;
  // Each stream's buffer is freed under that stream's mutex: a call that
  // holds the buffer finishes its launches first.
  for (hipStream_t st : streams) {
    std::lock_guard<std::mutex> stream_lock(stream_mutex(st));
    std::lock_guard<std::mutex> lock(g_ws_mu);
    auto it = g_ws.find(st);
    if (it == g_ws.end()) continue;
    if (it->second.ptr) {
      hipError_t e = hipStreamSynchronize(st);
      if (e == hipSuccess) e = hipFree(it->second.ptr);
      if (e != hipSuccess) rc = check_hip(e, "release_workspace");
    }
    g_ws.erase(it);
  }
  return rc;
}

}  // extern "C"
