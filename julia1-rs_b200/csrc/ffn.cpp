// j1_op_linear, j1_op_gated and their backward passes: argument checks, workspace layout and
// the launches. Everything here runs on the host. Device memory is only taken for operands whose
// rows do not start on 16-byte boundaries: the products read such an operand from a copy, in
// stream-ordered memory of the library's own pool (Copies below).
#include <atomic>
#include <climits>
#include <cstdint>
#include <mutex>
#include <string>

#include "ffn.h"
#include "model.h"

using namespace j1rt;

#define FFN_LAUNCH(expr, what)                                             \
  do {                                                                     \
    if (take_fault(J1_FAULT_LAUNCH)) return cuda_error(cudaErrorLaunchFailure, what " (injected)"); \
    const int rc_ = (expr);                                                \
    if (rc_) return cuda_error(static_cast<cudaError_t>(rc_), what);       \
  } while (0)

#define FFN_TRY(expr)          \
  do {                         \
    const j1_status s_ = (expr); \
    if (s_) return s_;         \
  } while (0)

namespace {

constexpr int kMaxDevices = 64;
constexpr int kMaxDim = 1 << 30;       // M, N, K
constexpr int kMaxGated = 1 << 29;     // N of a gated block: its two projections are rows of one product

// The operators' error word (0: no timed-out wait), one per device: a file-scope array, so that
// no call allocates (a call may be captured, or a pool may own all of the device's memory).
struct FfnDevice {
  std::atomic<bool> ready{false};
  int* err = nullptr;
  int num_sms = 0;
  cudaMemPool_t pool = nullptr;  // for operand copies
};
FfnDevice g_dev[kMaxDevices];
std::mutex g_dev_mutex;  // first use of a device; a failure leaves it for the next call

// The first CUDA call of a host thread may be one of these operators, and tensor maps can only be made with
// a context that is current: the runtime binds the device's when it is asked to.
cudaError_t bind_context(int dev) {
  using GetCurrent = CUresult (*)(CUcontext*);
  static const GetCurrent current = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    const cudaError_t e = cudaGetDriverEntryPoint("cuCtxGetCurrent", &fn, cudaEnableDefault, &found);
    return e == cudaSuccess && found == cudaDriverEntryPointSuccess ? reinterpret_cast<GetCurrent>(fn) : nullptr;
  }();
  CUcontext ctx = nullptr;
  if (current && current(&ctx) == CUDA_SUCCESS && ctx) return cudaSuccess;
  return cudaSetDevice(dev);
}

// The device's pool, which keeps what it has taken (as a model's workspace does).
cudaError_t make_pool(int dev, cudaMemPool_t* pool) {
  cudaMemPoolProps props = {};
  props.allocType = cudaMemAllocationTypePinned;
  props.location.type = cudaMemLocationTypeDevice;
  props.location.id = dev;
  cudaError_t e = cudaMemPoolCreate(pool, &props);
  if (e != cudaSuccess) return e;
  uint64_t keep = UINT64_MAX;
  e = cudaMemPoolSetAttribute(*pool, cudaMemPoolAttrReleaseThreshold, &keep);
  if (e != cudaSuccess) cudaMemPoolDestroy(*pool);
  return e;
}

// What the first use of a device prepares: kernels are loaded, whichever the calls will take, and the pool is made. A
// capture under way (this thread's, or another's in the global mode) would forbid that, and end: it touches no stream, so the
// thread takes the relaxed mode for it.
cudaError_t first_use(int dev, int** err, int* sms, cudaMemPool_t* pool) {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode);
  if (e != cudaSuccess) return e;
  e = ffn_error_word(err);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess) e = load_ffn_rows();
  if (e == cudaSuccess) e = load_ffn_tc_bf16();
  if (e == cudaSuccess) e = load_ffn_tc_fp16();
  if (e == cudaSuccess) e = make_pool(dev, pool);
  const cudaError_t back = cudaThreadExchangeStreamCaptureMode(&mode);
  if (e == cudaSuccess && back != cudaSuccess) cudaMemPoolDestroy(*pool);
  return e == cudaSuccess ? back : e;
}

j1_status device_state(FfnDevice** out, int* ordinal) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = bind_context(dev);
  if (e != cudaSuccess) return cuda_error(e, "cudaGetDevice");
  if (dev < 0 || dev >= kMaxDevices) return set_error(J1_ERR_UNSUPPORTED, "device ordinal above 63");
  FfnDevice& s = g_dev[dev];
  if (!s.ready.load(std::memory_order_acquire)) {
    std::lock_guard<std::mutex> lock(g_dev_mutex);
    if (!s.ready.load(std::memory_order_relaxed)) {  // else another thread was first: its values are in use
      int* err = nullptr;
      int sms = 0;
      cudaMemPool_t pool = nullptr;
      const cudaError_t rc = first_use(dev, &err, &sms, &pool);
      if (rc != cudaSuccess) {
        cudaGetLastError();
        return cuda_error(rc, "first use of the device");
      }
      s.pool = pool;
      s.err = err;
      s.num_sms = sms;
      s.ready.store(true, std::memory_order_release);
    }
  }
  *out = &s;
  *ordinal = dev;
  return J1_OK;
}

// One matrix (or vector) argument of a call.
struct Arg {
  const char* name;
  const void* p;
  int64_t rows, cols, ld;
  int elem;  // bytes
  bool write;
  uint64_t lo() const { return reinterpret_cast<uintptr_t>(p); }
  uint64_t hi() const {
    return rows && cols ? lo() + (static_cast<uint64_t>(rows - 1) * ld + cols) * elem : lo();
  }
};

j1_status bad(const std::string& msg) { return set_error(J1_ERR_INVALID_ARG, msg); }

// Whether two arguments share memory. Matrices of one row stride whose columns are apart (two
// halves of the rows of one buffer) do not, although their address ranges interleave.
bool overlap(const Arg& a, const Arg& b) {
  if (a.lo() >= b.hi() || b.lo() >= a.hi()) return false;
  if (a.ld != b.ld || a.elem != b.elem || a.rows < 2 || b.rows < 2) return true;
  const uint64_t row = static_cast<uint64_t>(a.ld) * a.elem;
  const uint64_t d = a.lo() <= b.lo() ? (b.lo() - a.lo()) % row : (row - (a.lo() - b.lo()) % row) % row;
  return d < static_cast<uint64_t>(a.cols) * a.elem || d + static_cast<uint64_t>(b.cols) * b.elem > row;
}

j1_status check_sizes(int M, int N, int K, int max_n) {
  if (M < 0 || N <= 0 || K <= 0) return bad("M must be >= 0, N and K positive");
  if (M > kMaxDim || N > kMaxDim || K > kMaxDim) return set_error(J1_ERR_UNSUPPORTED, "sizes above 2^30");
  if (N > max_n) return set_error(J1_ERR_UNSUPPORTED, "N above 2^29");
  return J1_OK;
}

// Host checks of a call's sizes and matrices: strides, alignment, overlaps. `same`: index of an
// input that the output `same_out` may coincide with.
j1_status check_args(int dtype, int act, int M, int N, int K, int max_n, const Arg* a, int n, int same = -1,
                     int same_out = -1) {
  if (dtype != J1_DTYPE_BF16 && dtype != J1_DTYPE_FP16) return bad("unknown dtype");
  if (act < J1_ACT_NONE || act > J1_ACT_SILU) return bad("unknown activation");
  FFN_TRY(check_sizes(M, N, K, max_n));
  for (int i = 0; i < n; ++i) {
    if (!a[i].p) continue;
    if (a[i].ld < a[i].cols) return bad(std::string(a[i].name) + ": row stride below the row's width");
    if (a[i].ld > (int64_t(1) << 38)) return set_error(J1_ERR_UNSUPPORTED, std::string(a[i].name) + ": row stride above 2^38");
    if (a[i].rows > 1 && a[i].ld > (int64_t(1) << 46) / (a[i].rows - 1))
      return set_error(J1_ERR_UNSUPPORTED, std::string(a[i].name) + ": more than 2^46 elements");
    if (a[i].lo() % a[i].elem) return bad(std::string(a[i].name) + ": not aligned to its element type");
  }
  for (int i = 0; i < n; ++i) {
    if (!a[i].p || !a[i].write) continue;
    for (int j = 0; j < n; ++j) {
      if (j == i || !a[j].p || (a[j].write && j < i)) continue;
      if (i == same_out && j == same && a[i].p == a[j].p && a[i].ld == a[j].ld) continue;
      if (overlap(a[i], a[j]))
        return bad(std::string(a[i].name) + " overlaps " + a[j].name);
    }
  }
  return J1_OK;
}

// Every pointer must be device memory of the current device.
j1_status check_device(const Arg* a, int n, int device) {
  for (int i = 0; i < n; ++i) {
    if (!a[i].p || !a[i].rows) continue;
    cudaPointerAttributes at;
    const cudaError_t e = cudaPointerGetAttributes(&at, a[i].p);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return cuda_error(e, a[i].name);
    }
    if (at.type != cudaMemoryTypeDevice) return bad(std::string(a[i].name) + " is not device memory");
    if (at.device != device)
      return bad(std::string(a[i].name) + " is on device " + std::to_string(at.device) + ", the current device is " +
                 std::to_string(device));
  }
  return J1_OK;
}

j1_status finish(FfnDevice* d, cudaStream_t st, int sync) {
  if (!sync) return J1_OK;
  cudaError_t e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return cuda_error(e, "op");
  int w = 0;
  e = cudaMemcpyAsync(&w, d->err, 4, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return cuda_error(e, "op error word");
  if (w) {
    e = cudaMemsetAsync(d->err, 0, 4, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    return set_error(J1_ERR_DEVICE_TIMEOUT, "device-side wait timed out (site " + std::to_string(w >> 16) + ")");
  }
  return J1_OK;
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

FfnGemm gemm_for(int dtype, int layout, int M, int N, int K, const FfnDevice* d) {
  FfnGemm g = {};
  g.fp16 = dtype == J1_DTYPE_FP16;
  g.layout = layout;
  g.act = J1_ACT_NONE;
  g.M = M, g.N = N, g.K = K;
  g.segs = 1;
  g.row1 = g.rows0 = INT_MAX;
  g.err = d->err;
  g.num_sms = d->num_sms;
  return g;
}

// Copies of a call's operands. TMA reads rows on 16-byte boundaries only; the products' other operands
// are copied first, all in one launch. (Reading them in the product instead, loader warps shifting
// aligned 16-byte pieces into place, kept the tensor cores waiting: 65536 x 771 x 1155 took 527-606 us,
// with the copies 198. A copy costs its bytes twice.) The memory is taken and given back in stream
// order: calls on several streams, and captured graphs, have their own.
class Copies {
 public:
  explicit Copies(cudaStream_t st) : st_(st) {}
  ~Copies() {
    if (mem_) cudaFreeAsync(mem_, st_);
  }
  Copies(const Copies&) = delete;
  Copies& operator=(const Copies&) = delete;

  // Notes the operands of a product that need it.
  void add(FfnGemm& g) {
    const int na = g.segs, nb = g.gated ? 2 : g.segs;
    for (int i = 0; i < na + nb; ++i) {
      const bool a = i < na;
      FfnMat& m = a ? g.a[i] : g.b[i - na];
      FfnCopy o = {};
      o.rows = a ? (g.layout == FFN_TN ? g.K : g.M) : (g.layout == FFN_NT ? g.N : g.K);
      o.cols = a ? (g.layout == FFN_TN ? g.M : g.K) : (g.layout == FFN_NT ? g.K : g.N);
      const long long ld = (static_cast<long long>(o.cols) + 7) / 8 * 8;
      if (o.rows == 1) m.ld = ld;  // one row: the stride is never used
      if (ffn_rows16(m)) continue;
      o.src = m;
      o.dst.ld = ld;
      operands_[c_.n] = &m;
      at_[c_.n] = bytes_;
      c_.m[c_.n++] = o;
      bytes_ += up256(static_cast<size_t>(o.rows) * ld * 2);
    }
  }
  // Makes the copies and puts them in their operands' places.
  j1_status make(FfnDevice* d) {
    if (!c_.n) return J1_OK;
    if (take_fault(J1_FAULT_ALLOC)) return set_error(J1_ERR_OOM, "operand copies: device allocation failed (injected)");
    const cudaError_t e = cudaMallocFromPoolAsync(&mem_, bytes_, d->pool, st_);
    if (e != cudaSuccess) {
      cudaGetLastError();
      mem_ = nullptr;
      return cuda_error(e, "operand copies");
    }
    for (int i = 0; i < c_.n; ++i) {
      c_.m[i].dst.p = static_cast<uint8_t*>(mem_) + at_[i];
      *operands_[i] = c_.m[i].dst;
    }
    FFN_LAUNCH(launch_ffn_copies(c_, st_), "operand copies");
    return J1_OK;
  }
  j1_status release() {
    void* mem = mem_;
    mem_ = nullptr;
    const cudaError_t e = mem ? cudaFreeAsync(mem, st_) : cudaSuccess;
    return e == cudaSuccess ? J1_OK : cuda_error(e, "operand copies");
  }

 private:
  cudaStream_t st_;
  FfnMat* operands_[4] = {};
  FfnCopies c_ = {};
  size_t bytes_ = 0, at_[4] = {};
  void* mem_ = nullptr;
};

// ---- backward workspace: gradients at the pre-activations (rows padded to 32 elements; the
// gated pair side by side), FP16's scale, slab sums of the bias gradients, partial products of dw.
int pad32(int n) { return (n + 31) / 32 * 32; }
// They are kept in two parts (the value cut to the type and what is left of it: 16 significant bits of BF16, 22 of
// FP16), whose products are summed in one accumulator, so that the results are rounded once as the formulas have
// it. With one part the relative error of dx and dw against 64 bits is 0.00235 for BF16 and not 0.00166, at 1 x 64
// gradients and at 65536 x 1152 alike (errors and sums both grow with the root of the number of terms), for half
// the products' operations: 65536 x 1152 x 768 gated 450 us against 940, 2048 x 768 x 1152 linear 17.8 against 24.8. Without
// an activation or with ReLU (linear) they are dout or 0: one part holds them.
struct Workspace {
  size_t grads, scale, sums, partials, bytes;  // offsets of the four parts, total
  size_t partial_bytes;
  long long ld, lo;  // of the gradients: row stride, distance of the second part
};
Workspace workspace_for(int M, int N, int K, int projections) {
  Workspace w;
  w.lo = static_cast<long long>(projections) * pad32(N);
  w.ld = 2 * w.lo;
  w.grads = 0;
  w.scale = up256(static_cast<size_t>(M) * w.ld * 2);
  w.sums = w.scale + up256(kFfnScaleFloats * sizeof(float));
  w.partials = w.sums + up256(static_cast<size_t>(ffn_grad_slabs(M, N)) * projections * N * 4);
  w.partial_bytes = ffn_partial_bytes(projections * pad32(N), K, M);
  w.bytes = w.partials + up256(w.partial_bytes);
  return w;
}

// The sizes of a backward pass's products (parts: the gradients at the pre-activations are in two): dx (a gated
// block's projections are two segments) and dw (their weights' rows are one product, the second's from pad32(N)).
FfnGemm dx_product(int dtype, int M, int N, int K, int projections, bool parts, const Workspace& ws, const FfnDevice* d) {
  FfnGemm g = gemm_for(dtype, FFN_NN, M, K, N, d);
  g.segs = projections;
  g.lo = parts ? ws.lo : 0;
  return g;
}
FfnGemm dw_product(int dtype, int M, int N, int K, int projections, bool parts, const Workspace& ws, void* workspace, const FfnDevice* d) {
  FfnGemm g = gemm_for(dtype, FFN_TN, projections == 2 ? pad32(N) + N : N, K, M, d);
  if (projections == 2) {
    g.rows0 = N;
    g.row1 = pad32(N);
  }
  g.lo = parts ? ws.lo : 0;
  g.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ws.partials);
  g.partial_bytes = ws.partial_bytes;
  return g;
}

j1_status workspace_query(int M, int N, int K, int projections, size_t* bytes) {
  if (!bytes) return bad("NULL argument");
  FFN_TRY(check_sizes(M, N, K, projections == 2 ? kMaxGated : kMaxDim));
  *bytes = workspace_for(M, N, K, projections).bytes;
  return J1_OK;
}

j1_status check_workspace(const void* p, size_t bytes, size_t need) {
  if (bytes < need || (need && !p))
    return bad("workspace of " + std::to_string(bytes) + " bytes, " + std::to_string(need) + " needed");
  if (reinterpret_cast<uintptr_t>(p) % 256) return bad("workspace must be 256-byte aligned");
  return J1_OK;
}

// The rest of a backward pass behind its row kernel: dx, and beside it the bias gradients' sums and the
// weights' gradients. Long products run one after the other: side by side their tails meet, but the second
// one's reads disturb the first one's in L2 (gradients in one part: 2 x 0.23 TFLOP, 65536 x 1152 x 768 gated, 452 us against 444; 2 x
// 0.06, 32768 x 768 x 1152, 119 against 120; 2 x 0.004, 2048 x 768 x 1152, 19.1 against 20.4).
j1_status backward_products(const FfnGrad& k, FfnGemm* dx, FfnGemm* dw, cudaStream_t st) {
  const bool sums = ffn_grad_sums(k);
  const bool lengthy = dx && 2.0 * dx->M * dx->N * dx->K * dx->segs * (dx->lo ? 2 : 1) > 1e11;
  const int apart = dx && !lengthy && (sums || dw);
  if (dx) {
    dx->late = apart;
    FFN_LAUNCH(launch_ffn_gemm(*dx, st), "dx launch");
  }
  if (sums) FFN_LAUNCH(launch_ffn_grad_sums(k, apart, st), "bias gradient launch");
  if (dw) {
    dw->early = apart;
    FFN_LAUNCH(launch_ffn_gemm(*dw, st), "dw launch");
  }
  return J1_OK;
}

j1_status zero_rows(void* p, int64_t ld, int rows, int cols, size_t elem, cudaStream_t st) {
  if (!p) return J1_OK;
  const cudaError_t e = cudaMemset2DAsync(p, ld * elem, 0, static_cast<size_t>(cols) * elem, rows, st);
  return e == cudaSuccess ? J1_OK : cuda_error(e, "memset");
}

}  // namespace

extern "C" {

j1_status j1_op_linear(const j1_linear_args* a, void* stream, int sync) {
  return guard("j1_op_linear", [&]() -> j1_status {
    if (!a || !a->w || (a->M > 0 && (!a->x || !a->out))) return bad("NULL argument");
    const Arg args[] = {{"x", a->x, a->M, a->K, a->ldx, 2, false},
                        {"w", a->w, a->N, a->K, a->ldw, 2, false},
                        {"bias", a->bias, 1, a->N, a->N, 4, false},
                        {"residual", a->residual, a->M, a->N, a->ldr, 2, false},
                        {"out", a->out, a->M, a->N, a->ldo, 2, true},
                        {"pre", a->pre, a->M, a->N, a->ldp, 2, true}};
    FFN_TRY(check_args(a->dtype, a->act, a->M, a->N, a->K, kMaxDim, args, 6, 3, 4));
    FfnDevice* d;
    int dev;
    FFN_TRY(device_state(&d, &dev));
    FFN_TRY(check_device(args, 6, dev));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->M) {
      FfnGemm g = gemm_for(a->dtype, FFN_NT, a->M, a->N, a->K, d);
      g.act = a->act;
      g.a[0] = {a->x, a->ldx};
      g.b[0] = {a->w, a->ldw};
      g.bias[0] = a->bias;
      g.residual = {a->residual, a->ldr};
      g.out[0] = {a->out, a->ldo};
      g.pre[0] = {a->pre, a->ldp};
      Copies copies(st);
      copies.add(g);
      FFN_TRY(copies.make(d));
      FFN_LAUNCH(launch_ffn_gemm(g, st), "linear launch");
      FFN_TRY(copies.release());
    }
    return finish(d, st, sync);
  });
}

j1_status j1_op_gated(const j1_gated_args* a, void* stream, int sync) {
  return guard("j1_op_gated", [&]() -> j1_status {
    if (!a || !a->wa || !a->wg || (a->M > 0 && (!a->x || !a->out))) return bad("NULL argument");
    if (!a->pre_a != !a->pre_g) return bad("pre_a and pre_g go together");
    const Arg args[] = {{"x", a->x, a->M, a->K, a->ldx, 2, false},
                        {"wa", a->wa, a->N, a->K, a->ldwa, 2, false},
                        {"wg", a->wg, a->N, a->K, a->ldwg, 2, false},
                        {"ba", a->ba, 1, a->N, a->N, 4, false},
                        {"bg", a->bg, 1, a->N, a->N, 4, false},
                        {"out", a->out, a->M, a->N, a->ldo, 2, true},
                        {"pre_a", a->pre_a, a->M, a->N, a->ldpa, 2, true},
                        {"pre_g", a->pre_g, a->M, a->N, a->ldpg, 2, true}};
    FFN_TRY(check_args(a->dtype, a->act, a->M, a->N, a->K, kMaxGated, args, 8));
    FfnDevice* d;
    int dev;
    FFN_TRY(device_state(&d, &dev));
    FFN_TRY(check_device(args, 8, dev));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->M) {
      FfnGemm g = gemm_for(a->dtype, FFN_NT, a->M, a->N, a->K, d);
      g.gated = 1;
      g.act = a->act;
      g.a[0] = {a->x, a->ldx};
      g.b[0] = {a->wa, a->ldwa};
      g.b[1] = {a->wg, a->ldwg};
      g.bias[0] = a->ba;
      g.bias[1] = a->bg;
      g.out[0] = {a->out, a->ldo};
      g.pre[0] = {a->pre_a, a->ldpa};
      g.pre[1] = {a->pre_g, a->ldpg};
      Copies copies(st);
      copies.add(g);
      FFN_TRY(copies.make(d));
      FFN_LAUNCH(launch_ffn_gemm(g, st), "gated launch");
      FFN_TRY(copies.release());
    }
    return finish(d, st, sync);
  });
}

j1_status j1_op_linear_backward_workspace(int32_t M, int32_t N, int32_t K, size_t* bytes) {
  return guard("j1_op_linear_backward_workspace", [&]() -> j1_status { return workspace_query(M, N, K, 1, bytes); });
}
j1_status j1_op_gated_backward_workspace(int32_t M, int32_t N, int32_t K, size_t* bytes) {
  return guard("j1_op_gated_backward_workspace", [&]() -> j1_status { return workspace_query(M, N, K, 2, bytes); });
}

j1_status j1_op_linear_backward(const j1_linear_grad_args* a, void* stream, int sync) {
  return guard("j1_op_linear_backward", [&]() -> j1_status {
    if (!a || (a->M > 0 && !a->dout)) return bad("NULL argument");
    if (!a->dx && !a->dw && !a->dbias && a->M > 0) return bad("no gradient wanted");
    if (a->dw && !a->x && a->M > 0) return bad("dw needs x");
    if (a->dx && !a->w) return bad("dx needs w");
    if (a->act != J1_ACT_NONE && !a->pre && a->M > 0) return bad("pre is NULL");
    const bool slope = a->act != J1_ACT_NONE;
    const Arg args[] = {{"dout", a->dout, a->M, a->N, a->lddo, 2, false},
                        {"x", a->dw ? a->x : nullptr, a->M, a->K, a->ldx, 2, false},
                        {"w", a->dx ? a->w : nullptr, a->N, a->K, a->ldw, 2, false},
                        {"pre", slope ? a->pre : nullptr, a->M, a->N, a->ldp, 2, false},
                        {"dx", a->dx, a->M, a->K, a->lddx, 2, true},
                        {"dw", a->dw, a->N, a->K, a->lddw, 2, true},
                        {"dbias", a->dbias, 1, a->N, a->N, 4, true},
                        {"workspace", a->workspace, 1, static_cast<int64_t>(a->workspace_bytes),
                         static_cast<int64_t>(a->workspace_bytes), 1, true}};
    FFN_TRY(check_args(a->dtype, a->act, a->M, a->N, a->K, kMaxDim, args, 8));
    const Workspace ws = workspace_for(a->M, a->N, a->K, 1);
    FFN_TRY(check_workspace(a->workspace, a->workspace_bytes, ws.bytes));
    FfnDevice* d;
    int dev;
    FFN_TRY(device_state(&d, &dev));
    FFN_TRY(check_device(args, 8, dev));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->M == 0) {
      FFN_TRY(zero_rows(a->dw, a->lddw, a->N, a->K, 2, st));
      FFN_TRY(zero_rows(a->dbias, a->N, 1, a->N, 4, st));
      return finish(d, st, sync);
    }
    uint8_t* base = static_cast<uint8_t*>(a->workspace);
    FfnMat dp = {a->dout, a->lddo};
    const bool products = a->dx || a->dw;
    const bool copy = products && (slope || !ffn_rows16(dp));  // both products read it
    if (copy) dp = {base + ws.grads, ws.ld};
    const bool parts = ffn_two_parts(false, a->act);
    FfnGemm gx = dx_product(a->dtype, a->M, a->N, a->K, 1, parts, ws, d);
    FfnGemm gw = dw_product(a->dtype, a->M, a->N, a->K, 1, parts, ws, base, d);
    FfnGrad k = {};
    Copies copies(st);
    if (products && parts && a->dtype == J1_DTYPE_FP16)
      gx.scale = gw.scale = k.scale = reinterpret_cast<float*>(base + ws.scale);
    if (a->dx) {
      gx.a[0] = dp;
      gx.b[0] = {a->w, a->ldw};
      gx.out[0] = {a->dx, a->lddx};
      copies.add(gx);
    }
    if (a->dw) {
      gw.a[0] = dp;
      gw.b[0] = {a->x, a->ldx};
      gw.out[0] = {a->dw, a->lddw};
      copies.add(gw);
    }
    FFN_TRY(copies.make(d));
    if (copy || a->dbias) {
      k.fp16 = a->dtype == J1_DTYPE_FP16;
      k.act = a->act;
      k.M = a->M, k.N = a->N;
      k.dout = {a->dout, a->lddo};
      k.p0 = {slope ? a->pre : nullptr, a->ldp};
      if (copy) k.d0 = dp;
      if (copy) k.lo = gx.lo;
      k.sum0 = a->dbias;
      k.partials = reinterpret_cast<float*>(base + ws.sums);
      FFN_LAUNCH(launch_ffn_grad(k, st), "linear gradient launch");
    }
    FFN_TRY(backward_products(k, a->dx ? &gx : nullptr, a->dw ? &gw : nullptr, st));
    FFN_TRY(copies.release());
    return finish(d, st, sync);
  });
}

j1_status j1_op_gated_backward(const j1_gated_grad_args* a, void* stream, int sync) {
  return guard("j1_op_gated_backward", [&]() -> j1_status {
    if (!a || (a->M > 0 && (!a->dout || !a->pre_a || !a->pre_g))) return bad("NULL argument");
    if (!a->dwa != !a->dwg) return bad("dwa and dwg go together");
    if (!a->dx && !a->dwa && !a->dba && !a->dbg && a->M > 0) return bad("no gradient wanted");
    if (a->dwa && !a->x && a->M > 0) return bad("dwa and dwg need x");
    if (a->dx && (!a->wa || !a->wg)) return bad("dx needs wa and wg");
    const Arg args[] = {{"dout", a->dout, a->M, a->N, a->lddo, 2, false},
                        {"x", a->dwa ? a->x : nullptr, a->M, a->K, a->ldx, 2, false},
                        {"wa", a->dx ? a->wa : nullptr, a->N, a->K, a->ldwa, 2, false},
                        {"wg", a->dx ? a->wg : nullptr, a->N, a->K, a->ldwg, 2, false},
                        {"pre_a", a->pre_a, a->M, a->N, a->ldpa, 2, false},
                        {"pre_g", a->pre_g, a->M, a->N, a->ldpg, 2, false},
                        {"dx", a->dx, a->M, a->K, a->lddx, 2, true},
                        {"dwa", a->dwa, a->N, a->K, a->lddwa, 2, true},
                        {"dwg", a->dwg, a->N, a->K, a->lddwg, 2, true},
                        {"dba", a->dba, 1, a->N, a->N, 4, true},
                        {"dbg", a->dbg, 1, a->N, a->N, 4, true},
                        {"workspace", a->workspace, 1, static_cast<int64_t>(a->workspace_bytes),
                         static_cast<int64_t>(a->workspace_bytes), 1, true}};
    FFN_TRY(check_args(a->dtype, a->act, a->M, a->N, a->K, kMaxGated, args, 12));
    const Workspace ws = workspace_for(a->M, a->N, a->K, 2);
    FFN_TRY(check_workspace(a->workspace, a->workspace_bytes, ws.bytes));
    FfnDevice* d;
    int dev;
    FFN_TRY(device_state(&d, &dev));
    FFN_TRY(check_device(args, 12, dev));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->M == 0) {
      FFN_TRY(zero_rows(a->dwa, a->lddwa, a->N, a->K, 2, st));
      FFN_TRY(zero_rows(a->dwg, a->lddwg, a->N, a->K, 2, st));
      FFN_TRY(zero_rows(a->dba, a->N, 1, a->N, 4, st));
      FFN_TRY(zero_rows(a->dbg, a->N, 1, a->N, 4, st));
      return finish(d, st, sync);
    }
    uint8_t* base = static_cast<uint8_t*>(a->workspace);
    const int np = pad32(a->N);
    FfnGrad k = {};
    k.fp16 = a->dtype == J1_DTYPE_FP16;
    k.gated = 1;
    k.act = a->act;
    k.M = a->M, k.N = a->N;
    k.dout = {a->dout, a->lddo};
    k.p0 = {a->pre_a, a->ldpa};
    k.p1 = {a->pre_g, a->ldpg};
    if (a->dx || a->dwa) {
      k.d0 = {base + ws.grads, ws.ld};
      k.d1 = {base + ws.grads + static_cast<size_t>(np) * 2, ws.ld};
      k.lo = ws.lo;
      if (k.fp16) k.scale = reinterpret_cast<float*>(base + ws.scale);
    }
    k.sum0 = a->dba;
    k.sum1 = a->dbg;
    k.partials = reinterpret_cast<float*>(base + ws.sums);
    const bool parts = ffn_two_parts(true, a->act);
    FfnGemm gx = dx_product(a->dtype, a->M, a->N, a->K, 2, parts, ws, d);
    FfnGemm gw = dw_product(a->dtype, a->M, a->N, a->K, 2, parts, ws, base, d);
    gx.scale = gw.scale = k.scale;
    Copies copies(st);
    if (a->dx) {
      gx.a[0] = k.d0;
      gx.a[1] = k.d1;
      gx.b[0] = {a->wa, a->ldwa};
      gx.b[1] = {a->wg, a->ldwg};
      gx.out[0] = {a->dx, a->lddx};
      copies.add(gx);
    }
    if (a->dwa) {
      gw.a[0] = k.d0;
      gw.b[0] = {a->x, a->ldx};
      gw.out[0] = {a->dwa, a->lddwa};
      gw.out[1] = {a->dwg, a->lddwg};
      copies.add(gw);
    }
    FFN_TRY(copies.make(d));
    FFN_LAUNCH(launch_ffn_grad(k, st), "gated gradient launch");
    FFN_TRY(backward_products(k, a->dx ? &gx : nullptr, a->dwa ? &gw : nullptr, st));
    FFN_TRY(copies.release());
    return finish(d, st, sync);
  });
}

j1_status j1_selftest_ffn_plan(int32_t product, int32_t act, int32_t M, int32_t N, int32_t K, int32_t num_sms, int32_t* plan) {
  return guard("j1_selftest_ffn_plan", [&]() -> j1_status {
    if (!plan || product < 0 || product > 5 || num_sms < 2) return bad("unknown product, fewer than two SMs, or NULL argument");
    const int projections = product == 1 || product > 3 ? 2 : 1;
    if (act < J1_ACT_NONE || act > J1_ACT_SILU) return bad("unknown activation");
    FFN_TRY(check_sizes(M, N, K, projections == 2 ? kMaxGated : kMaxDim));
    if (!M) return bad("no rows");
    FfnDevice d;
    d.num_sms = num_sms;
    const Workspace ws = workspace_for(M, N, K, projections);
    const bool parts = ffn_two_parts(projections == 2, act);
    FfnGemm g;
    if (product < 2) {
      g = gemm_for(J1_DTYPE_BF16, FFN_NT, M, N, K, &d);
      g.gated = product;
    } else if (product == 2 || product == 4) {
      g = dx_product(J1_DTYPE_BF16, M, N, K, projections, parts, ws, &d);
    } else {
      uint8_t any;  // not touched: a workspace is there
      g = dw_product(J1_DTYPE_BF16, M, N, K, projections, parts, ws, &any, &d);
    }
    ffn_plan(g, plan);
    return J1_OK;
  });
}

}  // extern "C"
