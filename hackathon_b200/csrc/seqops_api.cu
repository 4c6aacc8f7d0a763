// C ABI of the prompt-side operators (include/b2e.h): argument checks, then the
// launchers of norm_fp8.cu, fp8_gemm.cu, conv.cu and scan.cu.
#include <functional>
#include <initializer_list>
#include <mutex>

#include "../../include/b2e.h"
#include "seqops.cuh"

namespace b2e {
int abi_call(const std::function<void()>& f);
}

using namespace b2e;

// The operators' error word, one a device, in the library's device image: the
// calls take no buffer for it and allocate nothing.
static __device__ int g_seqops_err;

namespace {

constexpr int kMaxDevices = 64;
std::mutex g_mu;
int* g_err_ptr[kMaxDevices] = {};

// Every size within the 32-bit indices of the kernels.
void check_extents(std::initializer_list<long long> sizes) {
  for (const long long n : sizes) B2E_CHECK(n <= kMaxExtent, kErrInvalid, "sizes are at most 2^31 - 1024");
}

bool known(int t) { return t == kF32 || t == kBF16 || t == kF16; }

SeqPlan to_plan(const b2e_sequences* s, int rows) {
  SeqPlan p{};
  check_extents({rows, s ? s->tokens : 0});
  if (s == nullptr) {  // one token a sequence, row i in state row i
    p.seqs = p.tokens = p.state_rows = rows;
    p.longest = rows > 0 ? 1 : 0;
    return p;
  }
  B2E_CHECK(s->seqs >= 0 && s->tokens >= 0 && s->state_rows >= 0 && s->longest >= 0, kErrInvalid, "negative plan sizes");
  B2E_CHECK(s->seqs <= kMaxSeqs, kErrInvalid, "a plan has at most 2^30 sequences");
  B2E_CHECK(s->starts != nullptr || (s->tokens == s->seqs), kErrInvalid, "a plan without starts has one token a sequence");
  B2E_CHECK(s->slots != nullptr || s->seqs <= s->state_rows, kErrInvalid, "more sequences than state rows");
  B2E_CHECK(s->longest <= s->tokens, kErrInvalid, "the longest sequence has more tokens than the plan");
  p.starts = s->starts;
  p.slots = s->slots;
  p.order = s->order;
  p.seqs = s->seqs;
  p.tokens = s->tokens;
  p.state_rows = s->state_rows;
  p.longest = s->longest;
  return p;
}

ScanParams to_scan(const b2e_sequences* plan, const b2e_scan_args* a) {
  B2E_CHECK(a != nullptr, kErrInvalid, "null scan arguments");
  B2E_CHECK(a->rows >= 0 && a->heads > 0 && a->size > 0 && a->state > 0, kErrInvalid, "scan sizes must be positive");
  B2E_CHECK(a->state <= kScanMaxState, kErrInvalid, "mamba2_scan: state columns must be in 1..256");
  B2E_CHECK((long long)a->heads * a->size <= kMaxExtent && a->heads <= 65535, kErrInvalid, "mamba2_scan: too many channels");
  B2E_CHECK(known(a->dtype), kErrInvalid, "unknown dtype");
  ScanParams p{};
  p.plan = to_plan(plan, a->rows);
  B2E_CHECK(p.plan.tokens <= a->rows, kErrInvalid, "the plan has more tokens than the operands have rows");
  p.ssm = a->ssm;
  p.type = a->dtype;
  p.x = a->x; p.ldx = a->ldx;
  p.b = a->b; p.ldb = a->ldb;
  p.c = a->c; p.ldc = a->ldc;
  p.dt = a->dt; p.lddt = a->lddt;
  p.a = a->a;
  p.d = a->d;
  p.z = a->z; p.ldz = a->ldz;
  p.y = a->y; p.ldy = a->ldy;
  p.heads = a->heads;
  p.size = a->size;
  p.state = a->state;
  p.softplus = a->softplus != 0;
  return p;
}

}  // namespace

namespace b2e {
int* seqops_error_word() {
  int dev = 0;
  B2E_CUDA(cudaGetDevice(&dev));
  B2E_CHECK(dev >= 0 && dev < kMaxDevices, kErrInvalid, "device ordinal above 63");
  std::lock_guard<std::mutex> lock(g_mu);
  if (!g_err_ptr[dev]) {
    void* p = nullptr;
    B2E_CUDA(cudaGetSymbolAddress(&p, g_seqops_err));
    g_err_ptr[dev] = static_cast<int*>(p);
  }
  return g_err_ptr[dev];
}
}  // namespace b2e

extern "C" {

int b2e_seqops_device_error(int32_t* code) {
  return abi_call([&] {
    B2E_CHECK(code != nullptr, kErrInvalid, "null output");
    int* w = seqops_error_word();
    B2E_CUDA(cudaDeviceSynchronize());
    B2E_CUDA(cudaMemcpy(code, w, sizeof(int), cudaMemcpyDeviceToHost));
    if (*code != 0) B2E_CUDA(cudaMemset(w, 0, sizeof(int)));
  });
}

int b2e_rms_norm_fp8(const void* x, int32_t x_dtype, int64_t ldx, const void* residual, int32_t r_dtype, int64_t ldr,
                     const float* weight, float eps, int32_t rows, int32_t cols, void* q, int64_t ldq, float* scale,
                     void* total, void* normed, void* stream) {
  return abi_call([&] {
    B2E_CHECK(rows >= 0 && cols > 0, kErrInvalid, "rms_norm_fp8: bad sizes");
    check_extents({rows, cols});
    B2E_CHECK(known(x_dtype), kErrInvalid, "unknown dtype");
    B2E_CHECK(rows == 0 || (x && q && scale), kErrInvalid, "null operand");
    B2E_CHECK(!residual || r_dtype == x_dtype || r_dtype == kF32, kErrInvalid,
              "rms_norm_fp8: the residual has x's dtype or float32");
    B2E_CHECK(residual || !total, kErrInvalid, "rms_norm_fp8: total needs a residual");
    B2E_CHECK(ldx >= cols && ldq >= cols && (!residual || ldr >= cols), kErrInvalid, "a row stride is shorter than a row");
    RmsFp8Params p{x, x_dtype, ldx, residual, r_dtype, ldr, weight, eps, 1, rows, cols,
                   static_cast<uint8_t*>(q), ldq, scale, total, normed};
    rms_fp8(p, static_cast<cudaStream_t>(stream));
  });
}

int b2e_quantize_fp8(const void* x, int32_t x_dtype, int64_t ldx, int32_t rows, int32_t cols, void* q, int64_t ldq,
                     float* scale, void* stream) {
  return abi_call([&] {
    B2E_CHECK(rows >= 0 && cols > 0, kErrInvalid, "quantize_fp8: bad sizes");
    check_extents({rows, cols});
    B2E_CHECK(known(x_dtype), kErrInvalid, "unknown dtype");
    B2E_CHECK(rows == 0 || (x && q && scale), kErrInvalid, "null operand");
    B2E_CHECK(ldx >= cols && ldq >= cols, kErrInvalid, "a row stride is shorter than a row");
    RmsFp8Params p{x, x_dtype, ldx, nullptr, x_dtype, 0, nullptr, 0.f, 0, rows, cols,
                   static_cast<uint8_t*>(q), ldq, scale, nullptr, nullptr};
    rms_fp8(p, static_cast<cudaStream_t>(stream));
  });
}

int b2e_quantize_fp8_weight(const void* w, int32_t w_dtype, int64_t ldw, int32_t rows, int32_t cols, void* q, int64_t ldq,
                            float* scale, void* stream) {
  return abi_call([&] {
    B2E_CHECK(rows > 0 && cols > 0 && rows <= 65535 * kFp8Group, kErrInvalid, "quantize_fp8_weight: bad sizes");
    check_extents({cols});
    B2E_CHECK(known(w_dtype), kErrInvalid, "unknown dtype");
    B2E_CHECK(w && q && scale, kErrInvalid, "null operand");
    B2E_CHECK(ldw >= cols && ldq >= cols, kErrInvalid, "a row stride is shorter than a row");
    quantize_weight_fp8({w, w_dtype, ldw, rows, cols, static_cast<uint8_t*>(q), ldq, scale}, static_cast<cudaStream_t>(stream));
  });
}

int b2e_fp8_linear(const void* q, int64_t ldq, const float* scale, int32_t m, int32_t k, const void* wq, int64_t ldw,
                   const float* wscale, int32_t n, const float* bias, int32_t act, void* y, int32_t y_dtype, int64_t ldy,
                   void* stream) {
  return abi_call([&] {
    B2E_CHECK(m >= 0 && n > 0 && k > 0, kErrInvalid, "fp8_linear: bad sizes");
    check_extents({m, n, k});
    B2E_CHECK(known(y_dtype), kErrInvalid, "unknown dtype");
    B2E_CHECK(act == 0 || act == 1, kErrInvalid, "unknown activation");
    if (m == 0) return;
    B2E_CHECK(q && scale && wq && wscale && y, kErrInvalid, "null operand");
    B2E_CHECK(ldq >= k && ldw >= k && ldy >= n, kErrInvalid, "a row stride is shorter than a row");
    B2E_CHECK(ldq % 16 == 0 && ldw % 16 == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0 &&
                  (reinterpret_cast<uintptr_t>(wq) & 15) == 0,
              kErrInvalid, "fp8_linear: rows of q and wq start on 16-byte boundaries");
    fp8_gemm({static_cast<const uint8_t*>(q), ldq, scale, m, k, static_cast<const uint8_t*>(wq), ldw, wscale, n, bias, act, y,
              y_dtype, ldy, seqops_error_word()},
             static_cast<cudaStream_t>(stream));
  });
}

int b2e_causal_conv(const b2e_sequences* plan, float* window, const void* x, int32_t dtype, int64_t ldx, int32_t rows,
                    int32_t channels, const float* weight, const float* bias, int32_t taps, int32_t act, void* y,
                    int64_t ldy, void* stream) {
  return abi_call([&] {
    B2E_CHECK(rows >= 0 && channels > 0 && taps >= 2 && taps <= 4, kErrInvalid, "causal_conv: 2 to 4 taps, positive sizes");
    check_extents({channels});
    B2E_CHECK(known(dtype), kErrInvalid, "unknown dtype");
    B2E_CHECK(act == 0 || act == 1, kErrInvalid, "unknown activation");
    ConvParams p{};
    p.plan = to_plan(plan, rows);
    B2E_CHECK(p.plan.tokens <= rows, kErrInvalid, "the plan has more tokens than the operands have rows");
    if (p.plan.tokens == 0) return;
    B2E_CHECK(window && x && weight && y, kErrInvalid, "null operand");
    B2E_CHECK(ldx >= channels && ldy >= channels, kErrInvalid, "a row stride is shorter than a row");
    p.window = window;
    p.x = x; p.ldx = ldx;
    p.type = dtype;
    p.w = weight;
    p.bias = bias;
    p.channels = channels;
    p.taps = taps;
    p.silu = act;
    p.y = y; p.ldy = ldy;
    p.err = seqops_error_word();
    causal_conv(p, static_cast<cudaStream_t>(stream));
  });
}

int b2e_mamba2_scan_workspace(const b2e_sequences* plan, const b2e_scan_args* args, int64_t* bytes) {
  return abi_call([&] {
    B2E_CHECK(bytes != nullptr, kErrInvalid, "null output");
    *bytes = int64_t(scan_workspace(to_scan(plan, args)));
  });
}

int b2e_mamba2_scan(const b2e_sequences* plan, const b2e_scan_args* args, void* work, int64_t work_bytes, void* stream) {
  return abi_call([&] {
    ScanParams p = to_scan(plan, args);
    if (p.plan.tokens == 0) return;
    B2E_CHECK(p.ssm && p.x && p.b && p.c && p.dt && p.a && p.y, kErrInvalid, "null operand");
    const long long ch = (long long)p.heads * p.size;
    B2E_CHECK(p.ldx >= ch && p.ldy >= ch && (!p.z || p.ldz >= ch) && p.ldb >= p.state && p.ldc >= p.state && p.lddt >= p.heads,
              kErrInvalid, "a row stride is shorter than a row");
    B2E_CHECK((reinterpret_cast<uintptr_t>(p.ssm) & 15) == 0 || p.state % 4 != 0, kErrInvalid,
              "mamba2_scan: ssm starts on a 16-byte boundary");
    p.work = work;
    p.work_bytes = work ? size_t(work_bytes < 0 ? 0 : work_bytes) : 0;
    B2E_CHECK(p.work_bytes >= scan_workspace(p), kErrInvalid, "mamba2_scan: the workspace is too small");
    B2E_CHECK((reinterpret_cast<uintptr_t>(work) & 15) == 0, kErrInvalid, "mamba2_scan: the workspace starts on a 16-byte boundary");
    p.err = seqops_error_word();
    mamba2_scan(p, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
