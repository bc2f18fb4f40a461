// Eager training ops of the SpartonHead path in C++ (libsparton_torch.so): the head, the MLM
// transform before it and the SPLADE loss after it, each with its autograd in C++, calling the
// C ABI of libsparton_hip.so (include/sparton.h). The modules (SpartonHead,
// SpartonMLMTransform, splade_loss) use these when torch.compile is not tracing, so that a
// training step dispatches no Python per op in the forward or the backward. The
// reference-named torch.library ops (sparton::fused_sparton_fwd/bwd, ...) are defined in
// Python, with their fake kernels; they compute the same things through the same C ABI and
// serve torch.compile and direct callers.
//
//   sparton_eager::head_train(hidden, weight, bias?, mask) -> reps
//       the training forward (reps, int32 argmax and fp32 reps from one kernel) whose backward
//       writes dH, dW, dbias rounded once to the parameters' dtype (sparton_kernel.py:643-707)
//   sparton_eager::head_encode(hidden, weight, bias?, mask) -> reps   (no argmax, no autograd)
//   sparton_eager::head_train_autocast(hidden, weight, bias?, mask, weight_c, bias_c?, pad)
//       -> reps; weight_c/bias_c are the compute-dtype copies of the fp32 masters weight/bias
//       (D zero-padded by pad); the backward writes fp32 gradients straight to the masters
//   sparton_eager::mlm_transform(x, weight, dense_bias, ln_weight, ln_bias, eps) -> y
//   sparton_eager::mlm_transform_typed(the same, with the vectors in x's dtype)
//       LayerNorm(gelu(x W^T + b)) (training/model.py:14-40)
//   sparton_eager::splade_loss(q, d?, temperature, w_ce, w_l1, w_flops) -> out[6]
//       (total, CE, L1 q, L1 d, FLOPS q, FLOPS d)  (training/train.py:73-94, :164-197)
//   sparton_eager::attention(q, k, v, mask?, causal, scale) -> out   (a backbone layer's attention)
//   sparton_eager::layer_norm(x, residual?, weight, bias?, eps) -> y   LayerNorm(x + residual)
//   sparton_eager::preference_loss(q, pos, neg, ref_margin?, temperature, beta, smoothing) -> (loss, margin)
//   sparton_eager::{attention,layer_norm,preference}_{fwd,bwd}: their halves, which the torch.library
//       ops call; preference_margin: the margins alone
//
// The Python callers validate shapes and dtypes first (the same checks, and error types, as
// the torch.library ops); here only what the C ABI needs is enforced.
#include <ATen/ATen.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include <hipblaslt/hipblaslt.h>

#include <algorithm>
#include <cstring>
#include <mutex>
#include <unordered_map>

#include "../../include/sparton.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SPARTON_F32;
    case at::kBFloat16: return SPARTON_BF16;
    case at::kHalf: return SPARTON_F16;
    default: TORCH_CHECK(false, "sparton: unsupported dtype ", t);
  }
}

// The forward's dtype: fp32 follows torch's float32 matmul precision ('high' and 'medium':
// the bf16 hi/lo split, SPARTON_F32_SPLIT; 'highest': exact fp32), as the reference's GEMM
// does under the 'high' it sets at import (sparton_kernel.py:14).
int fwd_dtype_code(at::ScalarType t) {
  const int code = dtype_code(t);
  if (t == at::kFloat &&
      at::globalContext().float32MatmulPrecision() != at::Float32MatmulPrecision::HIGHEST)
    return code | SPARTON_F32_SPLIT;
  return code;
}

int mask_code(at::ScalarType t) {
  switch (t) {
    case at::kLong: return SPARTON_MASK_I64;
    case at::kInt: return SPARTON_MASK_I32;
    case at::kBool:
    case at::kByte: return SPARTON_MASK_U8;
    case at::kFloat: return SPARTON_MASK_F32;
    case at::kBFloat16: return SPARTON_MASK_BF16;
    case at::kHalf: return SPARTON_MASK_F16;
    default: TORCH_CHECK(false, "sparton: unsupported mask dtype ", t);
  }
}

void check(int rc, const char* what) {
  TORCH_CHECK(rc == SPARTON_OK, "sparton: ", what, " failed with status ", rc, ": ", sparton_strerror(rc));
}

void* stream_of(const Tensor& t) { return at::hip::getCurrentHIPStream(t.device().index()).stream(); }

// Row-major, unit inner stride, 16-byte aligned base (what the C ABI requires); undefined stays.
Tensor dense(const Tensor& t) {
  if (!t.defined()) return t;
  Tensor c = t.contiguous();
  if (reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 != 0) c = c.clone();
  return c;
}

const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* mptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor workspace(size_t bytes, const Tensor& like) {
  return at::empty({(int64_t)std::max<size_t>(bytes, 1)}, like.options().dtype(at::kByte));
}

// ---- the head --------------------------------------------------------------------------

struct FwdOut {
  Tensor reps, idx, reps32;
};

// sparton_fwd on dense tensors: reps in hidden's dtype, optionally the int32 argmax and fp32 reps.
FwdOut head_fwd(const Tensor& h, const Tensor& w, const Tensor& b, const Tensor& m, bool with_idx,
                bool with_f32) {
  const int64_t B = h.size(0), S = h.size(1), D = h.size(2), V = w.size(0);
  const int dt = fwd_dtype_code(h.scalar_type());
  FwdOut o;
  o.reps = at::empty({B, V}, h.options());
  if (with_idx) o.idx = at::empty({B, V}, h.options().dtype(at::kInt));
  if (with_f32) o.reps32 = at::empty({B, V}, h.options().dtype(at::kFloat));
  size_t ws_bytes = sparton_fwd_workspace_bytes(B, S, D, V, dt);
  Tensor ws;
  try {
    ws = workspace(ws_bytes, h);
  } catch (const c10::OutOfMemoryError&) {
    // the plan alone: larger fp32 batches then run without the bf16 parts of H and W
    const size_t least = sparton_fwd_workspace_min_bytes(B, S, D, V, dt);
    if (least == ws_bytes) throw;
    ws_bytes = least;
    ws = workspace(ws_bytes, h);
  }
  check(sparton_fwd(h.data_ptr(), w.data_ptr(), ptr(b), m.data_ptr(), mask_code(m.scalar_type()),
                    o.reps.data_ptr(), with_idx ? o.idx.data_ptr<int32_t>() : nullptr,
                    with_f32 ? o.reps32.data_ptr<float>() : nullptr, B, S, D, V, dt, ws.data_ptr(),
                    ws_bytes, stream_of(h)),
        "sparton_fwd");
  return o;
}

// sparton_bwd: gradients in `gdt` (fp32 or the inputs' dtype) from the fp32 reps.
std::tuple<Tensor, Tensor, Tensor> head_bwd(const Tensor& g, const Tensor& r32, const Tensor& idx,
                                            const Tensor& h, const Tensor& w, const Tensor& b,
                                            const Tensor& m, at::ScalarType gdt) {
  const int64_t B = h.size(0), S = h.size(1), D = h.size(2), V = w.size(0);
  const int dt = dtype_code(h.scalar_type());
  Tensor gd = dense(g.to(h.scalar_type()));
  Tensor dH = at::empty({B, S, D}, h.options().dtype(gdt));
  Tensor dW = at::empty({V, D}, h.options().dtype(gdt));
  Tensor db = at::empty({b.defined() ? V : 0}, h.options().dtype(gdt));
  const size_t ws_bytes = sparton_bwd_workspace_bytes(B, S, D, V);
  Tensor ws = workspace(ws_bytes, h);
  check(sparton_bwd(gd.data_ptr(), r32.data_ptr(), SPARTON_F32, idx.data_ptr<int32_t>(), m.data_ptr(),
                    mask_code(m.scalar_type()), h.data_ptr(), w.data_ptr(), dH.data_ptr(), dW.data_ptr(),
                    b.defined() ? db.data_ptr() : nullptr, dtype_code(gdt), ws.data_ptr(), ws_bytes, B, S,
                    D, V, dt, stream_of(h)),
        "sparton_bwd");
  return {dH, dW, db};
}

Tensor opt(const c10::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }

// torch::autograd::Function::apply records the metadata of every tensor argument, which an
// undefined tensor does not have: an absent optional goes in as an empty placeholder and a
// flag, and is undefined again inside.
Tensor present(const c10::optional<Tensor>& t, const Tensor& like) {
  return t.has_value() ? *t : at::empty({0}, like.options());
}

// (The operators below the head's pass another argument twice instead, which costs no allocation: its
// gradient at the absent place is undefined.)

// The forward's dispatch bodies: inference (no autograd) reps.
Tensor head_encode_cuda(const Tensor& hidden, const Tensor& weight, const c10::optional<Tensor>& bias,
                        const Tensor& mask) {
  c10::OptionalDeviceGuard guard(hidden.device());
  return head_fwd(dense(hidden), dense(weight), dense(opt(bias)), dense(mask), false, false).reps;
}

struct HeadTrainFn : public torch::autograd::Function<HeadTrainFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight,
                        const Tensor& bias_in, const Tensor& mask, bool has_bias) {
    at::AutoDispatchBelowADInplaceOrView below;
    c10::OptionalDeviceGuard guard(hidden.device());
    const Tensor bias = has_bias ? bias_in : Tensor();
    Tensor h = dense(hidden), w = dense(weight), b = dense(bias), m = dense(mask);
    FwdOut o = head_fwd(h, w, b, m, true, true);
    ctx->save_for_backward({o.reps32, o.idx, h, w, b, m});
    return o.reps;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    auto s = ctx->get_saved_variables();
    const Tensor& b = s[4];
    if (!grads[0].defined()) return variable_list(5);
    c10::OptionalDeviceGuard guard(s[2].device());
    auto [dH, dW, db] = head_bwd(grads[0], s[0], s[1], s[2], s[3], b, s[5], s[2].scalar_type());
    return {dH, dW, b.defined() ? db : Tensor(), Tensor(), Tensor()};
  }
};

Tensor head_train_autograd(const Tensor& hidden, const Tensor& weight, const c10::optional<Tensor>& bias,
                           const Tensor& mask) {
  return HeadTrainFn::apply(hidden, weight, present(bias, hidden), mask, bias.has_value());
}

// Mixed precision: hidden and the masters weight/bias are fp32; weight_c/bias_c are their
// compute-dtype copies (D zero-padded by pad). The forward casts hidden the same way; the
// backward asks the kernels for fp32 gradients, which go to the masters unrounded.
struct HeadAutocastFn : public torch::autograd::Function<HeadAutocastFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight,
                        const Tensor& bias_in, const Tensor& mask, const Tensor& weight_c,
                        const Tensor& bias_c_in, int64_t pad, bool has_bias) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor bias = has_bias ? bias_in : Tensor();
    const Tensor bias_c = has_bias ? bias_c_in : Tensor();
    c10::OptionalDeviceGuard guard(hidden.device());
    Tensor h = hidden.to(weight_c.scalar_type());
    if (pad > 0) h = at::constant_pad_nd(h, {0, pad});
    h = dense(h);
    Tensor w = dense(weight_c), b = dense(bias_c), m = dense(mask);
    FwdOut o = head_fwd(h, w, b, m, true, true);
    ctx->save_for_backward({o.reps32, o.idx, h, w, b, m});
    ctx->saved_data["D"] = hidden.size(-1);
    ctx->saved_data["hidden_dtype"] = static_cast<int64_t>(hidden.scalar_type());
    ctx->saved_data["has_bias"] = bias.defined();
    return o.reps;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(8);
    auto s = ctx->get_saved_variables();
    c10::OptionalDeviceGuard guard(s[2].device());
    auto [dH, dW, db] = head_bwd(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], at::kFloat);
    const int64_t D = ctx->saved_data["D"].toInt();
    if (dH.size(-1) != D) {  // drop the zero padding columns
      dH = dH.narrow(-1, 0, D);
      dW = dW.narrow(-1, 0, D);
    }
    const auto hdt = static_cast<at::ScalarType>(ctx->saved_data["hidden_dtype"].toInt());
    return {dH.to(hdt), dW, ctx->saved_data["has_bias"].toBool() ? db : Tensor(),
            Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor head_train_autocast_autograd(const Tensor& hidden, const Tensor& weight,
                                    const c10::optional<Tensor>& bias, const Tensor& mask,
                                    const Tensor& weight_c, const c10::optional<Tensor>& bias_c,
                                    int64_t pad) {
  TORCH_CHECK(bias.has_value() == bias_c.has_value(), "sparton: bias and its copy go together");
  return HeadAutocastFn::apply(hidden, weight, present(bias, hidden), mask, weight_c,
                               present(bias_c, weight_c), pad, bias.has_value());
}

// The CUDA-key bodies of the training ops, reached when no input needs a gradient (no
// autograd node is recorded): the reps alone.
Tensor head_train_cuda(const Tensor& hidden, const Tensor& weight, const c10::optional<Tensor>& bias,
                       const Tensor& mask) {
  return head_encode_cuda(hidden, weight, bias, mask);
}

Tensor head_train_autocast_cuda(const Tensor& hidden, const Tensor& weight,
                                const c10::optional<Tensor>& bias, const Tensor& mask,
                                const Tensor& weight_c, const c10::optional<Tensor>& bias_c, int64_t pad) {
  c10::OptionalDeviceGuard guard(hidden.device());
  Tensor h = hidden.to(weight_c.scalar_type());
  if (pad > 0) h = at::constant_pad_nd(h, {0, pad});
  return head_fwd(dense(h), dense(weight_c), dense(opt(bias_c)), dense(mask), false, false).reps;
}

// ---- cached hipBLASLt GEMMs (the transform's, 16-bit) ------------------------------------
//
// Column-major D[m x n] = op(A)[m x k] op(B)[k x n], fp32 accumulation, optionally a strided
// batch. torch's GEMM path asks hipBLASLt's heuristic for an algorithm on every call (~20 us of
// host time per GEMM); here the descriptors and the heuristic's first algorithm are made once
// per shape and device and kept, so a call is one hipblasLtMatmul. The library is the one
// torch loads (same soname), so the process holds one hipBLASLt.
struct GemmKey {
  int device, in_type, out_type, ta, tb, batch;
  int64_t m, n, k, lda, ldb, ldd, sa, sb, sd;
};
bool operator==(const GemmKey& x, const GemmKey& y) { return std::memcmp(&x, &y, sizeof(GemmKey)) == 0; }
struct GemmKeyHash {
  size_t operator()(const GemmKey& key) const {
    const unsigned char* p = reinterpret_cast<const unsigned char*>(&key);
    uint64_t h = 1469598103934665603ull;  // FNV-1a over the (zero-initialised) key bytes
    for (size_t i = 0; i < sizeof(GemmKey); ++i) h = (h ^ p[i]) * 1099511628211ull;
    return (size_t)h;
  }
};
struct GemmPlan {
  hipblasLtMatmulDesc_t op = nullptr;
  hipblasLtMatrixLayout_t a = nullptr, b = nullptr, d = nullptr;
  hipblasLtMatmulAlgo_t algo;
  size_t ws = 0;
};
constexpr int kMaxGemmDevices = 64;
constexpr uint64_t kGemmMaxWorkspace = (uint64_t)32 << 20;
std::mutex g_lt_mu;
hipblasLtHandle_t g_lt[kMaxGemmDevices] = {};
std::unordered_map<GemmKey, GemmPlan, GemmKeyHash> g_plans;

void lt_check(hipblasStatus_t st, const char* what) {
  TORCH_CHECK(st == HIPBLAS_STATUS_SUCCESS, "sparton: hipBLASLt ", what, " failed (status ", (int)st, ")");
}

GemmKey gemm_key(int device, hipDataType in, hipDataType out, bool ta, bool tb, int64_t m, int64_t n,
                 int64_t k, int64_t lda, int64_t ldb, int64_t ldd, int batch = 1, int64_t sa = 0,
                 int64_t sb = 0, int64_t sd = 0) {
  GemmKey key;
  std::memset(&key, 0, sizeof(key));  // the padding bytes take part in == and the hash
  key.device = device;
  key.in_type = (int)in;
  key.out_type = (int)out;
  key.ta = ta;
  key.tb = tb;
  key.batch = batch;
  key.m = m;
  key.n = n;
  key.k = k;
  key.lda = lda;
  key.ldb = ldb;
  key.ldd = ldd;
  key.sa = sa;
  key.sb = sb;
  key.sd = sd;
  return key;
}

// Called with the key's device current. The returned reference stays valid: the map only grows.
const GemmPlan& gemm_plan(const GemmKey& key, hipblasLtHandle_t* handle) {
  TORCH_CHECK(key.device >= 0 && key.device < kMaxGemmDevices, "sparton: device index out of range");
  std::lock_guard<std::mutex> lock(g_lt_mu);
  if (g_lt[key.device] == nullptr) lt_check(hipblasLtCreate(&g_lt[key.device]), "handle creation");
  *handle = g_lt[key.device];
  auto it = g_plans.find(key);
  if (it != g_plans.end()) return it->second;
  GemmPlan p;
  lt_check(hipblasLtMatmulDescCreate(&p.op, HIPBLAS_COMPUTE_32F, HIP_R_32F), "descriptor");
  const hipblasOperation_t ta = key.ta ? HIPBLAS_OP_T : HIPBLAS_OP_N;
  const hipblasOperation_t tb = key.tb ? HIPBLAS_OP_T : HIPBLAS_OP_N;
  lt_check(hipblasLtMatmulDescSetAttribute(p.op, HIPBLASLT_MATMUL_DESC_TRANSA, &ta, sizeof(ta)), "transA");
  lt_check(hipblasLtMatmulDescSetAttribute(p.op, HIPBLASLT_MATMUL_DESC_TRANSB, &tb, sizeof(tb)), "transB");
  const hipDataType in = (hipDataType)key.in_type, out = (hipDataType)key.out_type;
  lt_check(hipblasLtMatrixLayoutCreate(&p.a, in, key.ta ? key.k : key.m, key.ta ? key.m : key.k, key.lda), "layout A");
  lt_check(hipblasLtMatrixLayoutCreate(&p.b, in, key.tb ? key.n : key.k, key.tb ? key.k : key.n, key.ldb), "layout B");
  lt_check(hipblasLtMatrixLayoutCreate(&p.d, out, key.m, key.n, key.ldd), "layout D");
  if (key.batch > 1) {
    const int32_t bc = key.batch;
    const hipblasLtMatrixLayout_t lay[3] = {p.a, p.b, p.d};
    const int64_t str[3] = {key.sa, key.sb, key.sd};
    for (int i = 0; i < 3; ++i) {
      lt_check(hipblasLtMatrixLayoutSetAttribute(lay[i], HIPBLASLT_MATRIX_LAYOUT_BATCH_COUNT, &bc, sizeof(bc)), "batch");
      lt_check(hipblasLtMatrixLayoutSetAttribute(lay[i], HIPBLASLT_MATRIX_LAYOUT_STRIDED_BATCH_OFFSET, &str[i],
                                                 sizeof(str[i])), "batch stride");
    }
  }
  hipblasLtMatmulPreference_t pref = nullptr;
  lt_check(hipblasLtMatmulPreferenceCreate(&pref), "preference");
  lt_check(hipblasLtMatmulPreferenceSetAttribute(pref, HIPBLASLT_MATMUL_PREF_MAX_WORKSPACE_BYTES, &kGemmMaxWorkspace,
                                                 sizeof(kGemmMaxWorkspace)), "workspace preference");
  hipblasLtMatmulHeuristicResult_t res[1];
  int got = 0;
  const hipblasStatus_t hs = hipblasLtMatmulAlgoGetHeuristic(*handle, p.op, p.a, p.b, p.d, p.d, pref, 1, res, &got);
  hipblasLtMatmulPreferenceDestroy(pref);
  lt_check(hs, "heuristic");
  TORCH_CHECK(got > 0, "sparton: hipBLASLt found no algorithm for a ", key.m, " x ", key.n, " x ", key.k, " GEMM");
  p.algo = res[0].algo;
  p.ws = res[0].workspaceSize;
  return g_plans.emplace(key, p).first->second;
}

void lt_gemm(const GemmKey& key, const void* A, const void* B, void* D, const Tensor& like) {
  hipblasLtHandle_t handle = nullptr;
  const GemmPlan& p = gemm_plan(key, &handle);
  Tensor ws = workspace(p.ws, like);
  const float alpha = 1.0f, beta = 0.0f;
  lt_check(hipblasLtMatmul(handle, p.op, &alpha, A, p.a, B, p.b, &beta, D, p.d, D, p.d, &p.algo,
                           p.ws ? ws.data_ptr() : nullptr, p.ws, (hipStream_t)stream_of(like)),
           "matmul");
}

hipDataType lt_type(at::ScalarType t) { return t == at::kBFloat16 ? HIP_R_16BF : HIP_R_16F; }
bool lt_gemm_ok(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }

// z[M, Dout] = x2[M, Din] W[Dout, Din]^T (column-major: z^T = op_T(W) x2^T).
Tensor lt_linear(const Tensor& x2, const Tensor& w) {
  const int64_t M = x2.size(0), Din = x2.size(1), Dout = w.size(0);
  Tensor z = at::empty({M, Dout}, x2.options());
  lt_gemm(gemm_key(x2.get_device(), lt_type(x2.scalar_type()), lt_type(x2.scalar_type()), true, false, Dout, M, Din,
                   Din, Din, Dout),
          w.data_ptr(), x2.data_ptr(), z.data_ptr(), x2);
  return z;
}

// dx[M, Din] = dz[M, Dout] W[Dout, Din] (column-major: dx^T = W^T dz^T, both as stored).
Tensor lt_dgrad(const Tensor& dz, const Tensor& w) {
  const int64_t M = dz.size(0), Dout = dz.size(1), Din = w.size(1);
  Tensor dx = at::empty({M, Din}, dz.options());
  lt_gemm(gemm_key(dz.get_device(), lt_type(dz.scalar_type()), lt_type(dz.scalar_type()), false, false, Din, M, Dout,
                   Din, Dout, Din),
          w.data_ptr(), dz.data_ptr(), dx.data_ptr(), dz);
  return dx;
}

// ---- the MLM transform -------------------------------------------------------------------

// Row chunks of the transform's batched weight-gradient GEMM, or 0 for one plain GEMM (the same
// rule as sparton_amd/transform.py's _wgrad_chunks).
int64_t wgrad_chunks(int64_t M, int64_t D, at::ScalarType dt) {
  if ((dt != at::kBFloat16 && dt != at::kHalf) || M < 2048 || D % 64 != 0) return 0;
  const int64_t C = M <= 4096 ? 4 : (M <= 16384 ? 8 : 16);
  return M % (C * 64) == 0 ? C : 0;
}

// dW = dz^T x2: row chunks transposed by HIP, one batched GEMM with fp32 outputs, the chunk
// products summed in order and rounded once by HIP (transform.py's _weight_grad).
// For 16-bit, the chunks go to hipBLASLt as one strided batch over row chunks of dz and x2 as
// they lie (dz transposed by the GEMM's op flag, so no transpose kernel): chunk i's fp32
// product is column-major (Din x Dout), i.e. row-major dW [Dout][Din].
Tensor transform_weight_grad(const Tensor& dz, const Tensor& x2, int64_t M, int64_t D) {
  const int64_t C = wgrad_chunks(M, D, dz.scalar_type());
  if (C == 0) {
    if (!lt_gemm_ok(dz)) return at::mm(dz.t(), x2);
    Tensor dw = at::empty({D, D}, dz.options());  // column-major dW^T = x2^T dz
    lt_gemm(gemm_key(dz.get_device(), lt_type(dz.scalar_type()), lt_type(dz.scalar_type()), false, true, D, D, M,
                     D, D, D),
            x2.data_ptr(), dz.data_ptr(), dw.data_ptr(), dz);
    return dw;
  }
  const int code = dtype_code(dz.scalar_type());
  void* st = stream_of(dz);
  const int64_t Mc = M / C;
  Tensor part = at::empty({C, D, D}, dz.options().dtype(at::kFloat));
  lt_gemm(gemm_key(dz.get_device(), lt_type(dz.scalar_type()), HIP_R_32F, false, true, D, D, Mc, D, D, D, (int)C,
                   Mc * D, Mc * D, D * D),
          x2.data_ptr(), dz.data_ptr(), part.data_ptr(), dz);
  Tensor dw = at::empty({D, D}, dz.options());
  check(sparton_transform_chunk_sum(part.data_ptr<float>(), dw.data_ptr(), C, D * D, code, st),
        "sparton_transform_chunk_sum");
  return dw;
}

struct TransformFn : public torch::autograd::Function<TransformFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                        const Tensor& dense_bias, const Tensor& ln_weight, const Tensor& ln_bias,
                        double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    c10::OptionalDeviceGuard guard(x.device());
    const int64_t D = x.size(-1);
    Tensor x2 = x.reshape({-1, D});
    // hipBLASLt: cached plans for 16-bit, torch's F.linear otherwise
    Tensor z = lt_gemm_ok(x2) ? lt_linear(dense(x2), dense(weight)) : at::linear(x2, weight);
    const int64_t M = z.size(0);
    Tensor y = at::empty_like(z);
    Tensor mean = at::empty({M}, x.options().dtype(at::kFloat));
    Tensor rstd = at::empty({M}, x.options().dtype(at::kFloat));
    Tensor vb = dense(dense_bias), vg = dense(ln_weight), vt = dense(ln_bias);
    // 16-bit vectors are the module's parameters themselves: the backward takes the copies that the
    // kernel leaves, so that the parameters may change before it, as float32 copies of them did.
    Tensor kept = vb.scalar_type() == at::kFloat ? Tensor() : at::empty({2, D}, vb.options());
    check(sparton_transform_fwd_keep(z.data_ptr(), vb.data_ptr(), vg.data_ptr(), vt.data_ptr(),
                                     dtype_code(vb.scalar_type()), (float)eps, y.data_ptr(),
                                     mean.data_ptr<float>(), rstd.data_ptr<float>(), mptr(kept), M, D,
                                     dtype_code(x.scalar_type()), stream_of(x)),
          "sparton_transform_fwd");
    if (kept.defined()) ctx->save_for_backward({x, weight, z, kept, Tensor(), mean, rstd});
    else ctx->save_for_backward({x, weight, z, vb, vg, mean, rstd});
    return y.view(x.sizes());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(6);
    auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &weight = s[1], &z = s[2], &vb = s[3], &vg = s[4], &mean = s[5], &rstd = s[6];
    c10::OptionalDeviceGuard guard(x.device());
    const int64_t D = x.size(-1);
    Tensor x2 = x.reshape({-1, D});
    const int64_t M = x2.size(0);
    Tensor dy2 = grads[0].reshape({-1, D}).to(x.scalar_type()).contiguous();
    Tensor dz = at::empty_like(z);
    const void* bias = vb.data_ptr();
    const void* gamma = vg.defined() ? vg.data_ptr()  // or [2][D]: both
                                     : static_cast<const char*>(bias) + D * vb.element_size();
    Tensor dg = at::empty({D}, vb.options());
    Tensor dbt = at::empty_like(dg), dbd = at::empty_like(dg);
    const size_t ws_bytes = sparton_transform_workspace_bytes(M, D);
    Tensor ws = workspace(ws_bytes, x);
    check(sparton_transform_bwd_typed(dy2.data_ptr(), z.data_ptr(), bias, gamma,
                                      dtype_code(vb.scalar_type()), mean.data_ptr<float>(),
                                      rstd.data_ptr<float>(), dz.data_ptr(), dg.data_ptr(), dbt.data_ptr(),
                                      dbd.data_ptr(), ws.data_ptr(), ws_bytes, M, D,
                                      dtype_code(x.scalar_type()), stream_of(x)),
          "sparton_transform_bwd");
    Tensor dx = lt_gemm_ok(dz) ? lt_dgrad(dz, dense(weight)) : at::mm(dz, weight);
    Tensor dw = transform_weight_grad(dz, lt_gemm_ok(dz) ? dense(x2) : x2, M, D);
    return {dx.view(x.sizes()), dw, dbd, dg, dbt, Tensor()};
  }
};

// The vectors' dtype: float32 (mlm_transform), or x's own (mlm_transform_typed).
void check_vectors(const Tensor& b, const Tensor& g, const Tensor& t, at::ScalarType dt, const char* op) {
  TORCH_CHECK(b.scalar_type() == dt && g.scalar_type() == dt && t.scalar_type() == dt, "sparton: ", op,
              " takes its bias and LayerNorm vectors in ", dt);
}

Tensor transform_autograd(const Tensor& x, const Tensor& weight, const Tensor& dense_bias,
                          const Tensor& ln_weight, const Tensor& ln_bias, double eps) {
  check_vectors(dense_bias, ln_weight, ln_bias, at::kFloat, "mlm_transform");
  return TransformFn::apply(x, weight, dense_bias, ln_weight, ln_bias, eps);
}
Tensor transform_typed_autograd(const Tensor& x, const Tensor& weight, const Tensor& dense_bias,
                                const Tensor& ln_weight, const Tensor& ln_bias, double eps) {
  check_vectors(dense_bias, ln_weight, ln_bias, x.scalar_type(), "mlm_transform_typed");
  return TransformFn::apply(x, weight, dense_bias, ln_weight, ln_bias, eps);
}

Tensor transform_run(const Tensor& x, const Tensor& weight, const Tensor& dense_bias,
                     const Tensor& ln_weight, const Tensor& ln_bias, double eps) {
  c10::OptionalDeviceGuard guard(x.device());
  const int64_t D = x.size(-1);
  Tensor x2 = x.reshape({-1, D});
  Tensor z = lt_gemm_ok(x2) ? lt_linear(dense(x2), dense(weight)) : at::linear(x2, weight);
  const int64_t M = z.size(0);
  Tensor y = at::empty_like(z);
  Tensor mean = at::empty({M}, x.options().dtype(at::kFloat)), rstd = at::empty_like(mean);
  Tensor vb = dense(dense_bias), vg = dense(ln_weight), vt = dense(ln_bias);
  check(sparton_transform_fwd_typed(z.data_ptr(), vb.data_ptr(), vg.data_ptr(), vt.data_ptr(),
                                    dtype_code(vb.scalar_type()), (float)eps, y.data_ptr(),
                                    mean.data_ptr<float>(), rstd.data_ptr<float>(), M, D,
                                    dtype_code(x.scalar_type()), stream_of(x)),
        "sparton_transform_fwd");
  return y.view(x.sizes());
}
Tensor transform_cuda(const Tensor& x, const Tensor& weight, const Tensor& dense_bias,
                      const Tensor& ln_weight, const Tensor& ln_bias, double eps) {
  check_vectors(dense_bias, ln_weight, ln_bias, at::kFloat, "mlm_transform");
  return transform_run(x, weight, dense_bias, ln_weight, ln_bias, eps);
}
Tensor transform_typed_cuda(const Tensor& x, const Tensor& weight, const Tensor& dense_bias,
                            const Tensor& ln_weight, const Tensor& ln_bias, double eps) {
  check_vectors(dense_bias, ln_weight, ln_bias, x.scalar_type(), "mlm_transform_typed");
  return transform_run(x, weight, dense_bias, ln_weight, ln_bias, eps);
}

// ---- the SPLADE loss ----------------------------------------------------------------------

std::tuple<Tensor, Tensor> loss_fwd(const Tensor& q, const Tensor& d, double T, double w_ce,
                                    double w_l1, double w_flops) {
  const int64_t Bq = q.size(0), V = q.size(1), Bd = d.defined() ? d.size(0) : 0;
  Tensor out = at::empty({6}, q.options().dtype(at::kFloat));
  Tensor probs = at::empty({Bq, Bd}, q.options().dtype(at::kFloat));
  const size_t ws_bytes = sparton_loss_workspace_bytes(Bq, Bd, V);
  Tensor ws = workspace(ws_bytes, q);
  check(sparton_loss_fwd(q.data_ptr(), ptr(d), Bq, Bd, V, (float)T, (float)w_ce, (float)w_l1,
                         (float)w_flops, out.data_ptr<float>(), Bd ? probs.data_ptr<float>() : nullptr,
                         ws.data_ptr(), ws_bytes, dtype_code(q.scalar_type()), stream_of(q)),
        "sparton_loss_fwd");
  return {out, probs};
}

// The six terms (total, CE, L1(q), L1(d), FL(q), FL(d)) as separate scalars (views of the
// kernel's one output buffer), so that a caller backpropagating some of them (usually
// `total`) hands the backward only those gradients: the others stay undefined (no
// materialised zeros, no stack of six) and reach the kernel as NULL pointers.
using Loss6 = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;
Loss6 split6(const Tensor& out) {
  return {out.select(0, 0), out.select(0, 1), out.select(0, 2), out.select(0, 3), out.select(0, 4),
          out.select(0, 5)};
}

struct LossFn : public torch::autograd::Function<LossFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q_in, const Tensor& d_in, bool has_d,
                               double T, double w_ce, double w_l1, double w_flops) {
    at::AutoDispatchBelowADInplaceOrView below;
    c10::OptionalDeviceGuard guard(q_in.device());
    Tensor q = q_in.contiguous(), d = has_d ? d_in.contiguous() : Tensor();
    auto [out, probs] = loss_fwd(q, d, T, w_ce, w_l1, w_flops);
    ctx->save_for_backward({q, d, probs});
    ctx->saved_data["w_ce"] = w_ce;
    ctx->saved_data["w_l1"] = w_l1;
    ctx->saved_data["w_flops"] = w_flops;
    ctx->set_materialize_grads(false);
    auto t = split6(out);
    return {std::get<0>(t), std::get<1>(t), std::get<2>(t), std::get<3>(t), std::get<4>(t), std::get<5>(t)};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const float* gp[6];
    std::vector<Tensor> keep;
    bool any = false;
    for (int k = 0; k < 6; ++k) {
      gp[k] = nullptr;
      if (grads[k].defined()) {
        keep.push_back(grads[k].to(at::kFloat).contiguous());
        gp[k] = keep.back().data_ptr<float>();
        any = true;
      }
    }
    if (!any) return variable_list(7);
    auto s = ctx->get_saved_variables();
    const Tensor &q = s[0], &d = s[1], &probs = s[2];
    c10::OptionalDeviceGuard guard(q.device());
    const int64_t Bq = q.size(0), V = q.size(1), Bd = d.defined() ? d.size(0) : 0;
    Tensor dq = at::empty_like(q);
    Tensor dd = d.defined() ? at::empty_like(d) : Tensor();
    check(sparton_loss_bwd_terms(q.data_ptr(), ptr(d), Bd ? probs.data_ptr<float>() : nullptr, gp, Bq, Bd,
                                 V, (float)ctx->saved_data["w_ce"].toDouble(),
                                 (float)ctx->saved_data["w_l1"].toDouble(),
                                 (float)ctx->saved_data["w_flops"].toDouble(), dq.data_ptr(), mptr(dd),
                                 dtype_code(q.scalar_type()), stream_of(q)),
          "sparton_loss_bwd_terms");
    return {dq, dd, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Loss6 loss_autograd(const Tensor& q, const c10::optional<Tensor>& d, double T, double w_ce, double w_l1,
                    double w_flops) {
  auto o = LossFn::apply(q, present(d, q), d.has_value(), T, w_ce, w_l1, w_flops);
  return {o[0], o[1], o[2], o[3], o[4], o[5]};
}

Loss6 loss_cuda(const Tensor& q, const c10::optional<Tensor>& d, double T, double w_ce, double w_l1,
                double w_flops) {
  c10::OptionalDeviceGuard guard(q.device());
  Tensor dd = d.has_value() ? d->contiguous() : Tensor();
  return split6(std::get<0>(loss_fwd(q.contiguous(), dd, T, w_ce, w_l1, w_flops)));
}

// A backward's results where the caller keeps a graph of them (create_graph): the kernels have no
// second derivative, so that graph raises when it is run, instead of losing a term.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  const auto current = torch::autograd::get_current_node();  // none where grad_fn is called by hand
  torch::autograd::edge_list inputs;                         // the forward's
  if (current != nullptr) inputs = current->next_edges();
  auto node = std::make_shared<torch::autograd::Error>("sparton: gradients of this operator cannot be differentiated "
                                                       "again", std::move(inputs));
  for (Tensor& g : grads) {
    if (!g.defined()) continue;
    g = g.detach();
    torch::autograd::set_history(g, node);
  }
  return grads;
}

// ---- attention ----------------------------------------------------------------------------

// [B, H, S, D] with unit inner stride and rows that start on 16 bytes, as the C ABI reads it: the
// tensor itself where it is so (a view of a projection's output, or of a cache), else a copy. A head
// size that is not a multiple of 16 bytes is padded with zero columns, which change no product.
Tensor attention_rows(const Tensor& t) {
  const int64_t unit = 16 / t.element_size(), pad = (unit - t.size(3) % unit) % unit;
  if (pad > 0) return at::constant_pad_nd(t, {0, pad}).contiguous();  // heads innermost would stay so
  bool ok = t.stride(3) == 1 || t.size(3) == 1;
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) <= 1 || (t.stride(i) % unit == 0 && t.stride(i) >= 0));
  Tensor c = ok ? t : t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 != 0 ? c.clone(at::MemoryFormat::Contiguous) : c;
}

// [B, S, H, D] in memory, as the projection behind it reads it, seen as [B, H, S, D].
Tensor attention_like(const Tensor& t) {
  const int64_t B = t.size(0), H = t.size(1), S = t.size(2), D = t.size(3);
  return at::empty_strided({B, H, S, D}, {S * H * D, D, H * D, 1}, t.options());
}

void set_strides(int64_t* to, const Tensor& t) {
  for (int i = 0; i < 3; ++i) to[i] = t.stride(i);
}

sparton_attention_desc attention_desc(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& mask,
                                      const Tensor& out, bool causal, double scale) {
  sparton_attention_desc d;
  std::memset(&d, 0, sizeof(d));
  d.B = q.size(0);
  d.Hq = q.size(1);
  d.Hk = k.size(1);
  d.Sq = q.size(2);
  d.Sk = k.size(2);
  d.D = q.size(3);
  set_strides(d.q, q);
  set_strides(d.k, k);
  set_strides(d.v, v);
  set_strides(d.o, out);
  d.scale = (float)scale;
  d.causal = causal;
  d.dtype = dtype_code(q.scalar_type());
  if (mask.defined()) {
    d.mask_batch = mask.stride(0);
    d.mask_dtype = mask_code(mask.scalar_type());
  }
  return d;
}

// The mask [B, Sk] with unit inner stride (a row may be shared: stride 0 of an expanded batch).
Tensor attention_mask(const c10::optional<Tensor>& m) {
  if (!m.has_value()) return Tensor();
  return m->size(1) <= 1 || m->stride(1) == 1 ? *m : m->contiguous();
}

// out on the rows as they are (padded head size), and the rows' log sums if asked for.
std::tuple<Tensor, Tensor> attention_run(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& mask,
                                         bool causal, double scale, bool with_lse) {
  Tensor out = attention_like(q);
  Tensor lse = with_lse ? at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat)) : Tensor();
  const sparton_attention_desc d = attention_desc(q, k, v, mask, out, causal, scale);
  const size_t ws_bytes = sparton_attention_workspace_bytes(&d);
  Tensor ws = ws_bytes > 0 ? workspace(ws_bytes, q) : Tensor();  // seldom needed; an allocation costs the host 1.4 us
  check(sparton_attention_fwd(&d, q.data_ptr(), k.data_ptr(), v.data_ptr(), ptr(mask), out.data_ptr(),
                              with_lse ? lse.data_ptr<float>() : nullptr, mptr(ws), ws_bytes, stream_of(q)),
        "sparton_attention_fwd");
  return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor> attention_grads(const Tensor& dout, const Tensor& q, const Tensor& k,
                                                   const Tensor& v, const Tensor& mask, const Tensor& out,
                                                   const Tensor& lse, bool causal, double scale) {
  Tensor go = attention_rows(dout.to(q.scalar_type()));
  Tensor dq = attention_like(q), dk = attention_like(k), dv = attention_like(v);
  sparton_attention_desc d = attention_desc(q, k, v, mask, out, causal, scale);
  set_strides(d.d_o, go);
  set_strides(d.d_q, dq);
  set_strides(d.d_k, dk);
  set_strides(d.d_v, dv);
  const size_t ws_bytes = sparton_attention_bwd_workspace_bytes(&d);
  Tensor ws = workspace(ws_bytes, q);
  check(sparton_attention_bwd(&d, q.data_ptr(), k.data_ptr(), v.data_ptr(), ptr(mask), out.data_ptr(),
                              lse.data_ptr<float>(), go.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                              ws.data_ptr(), ws_bytes, stream_of(q)),
        "sparton_attention_bwd");
  return {dq, dk, dv};
}

Tensor head_cols(const Tensor& t, int64_t D) { return t.size(3) == D ? t : t.narrow(3, 0, D); }

// The pair that the torch.library ops run on (sparton::attention_fwd / _bwd).
std::tuple<Tensor, Tensor> attention_fwd_cuda(const Tensor& q, const Tensor& k, const Tensor& v,
                                              const c10::optional<Tensor>& mask, bool causal, double scale) {
  c10::OptionalDeviceGuard guard(q.device());
  auto [out, lse] = attention_run(attention_rows(q), attention_rows(k), attention_rows(v), attention_mask(mask),
                                  causal, scale, true);
  return {head_cols(out, q.size(3)), lse};
}
std::tuple<Tensor, Tensor, Tensor> attention_bwd_cuda(const Tensor& dout, const Tensor& q, const Tensor& k,
                                                      const Tensor& v, const c10::optional<Tensor>& mask,
                                                      const Tensor& out, const Tensor& lse, bool causal,
                                                      double scale) {
  c10::OptionalDeviceGuard guard(q.device());
  auto [dq, dk, dv] = attention_grads(dout, attention_rows(q), attention_rows(k), attention_rows(v),
                                      attention_mask(mask), attention_rows(out), lse, causal, scale);
  const int64_t D = q.size(3);
  return {head_cols(dq, D), head_cols(dk, D), head_cols(dv, D)};
}

struct AttentionFn : public torch::autograd::Function<AttentionFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                        const Tensor& mask_in, bool has_mask, bool causal, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    c10::OptionalDeviceGuard guard(q_in.device());
    Tensor q = attention_rows(q_in), k = attention_rows(k_in), v = attention_rows(v_in);
    Tensor mask = has_mask ? attention_mask(mask_in) : Tensor();
    auto [out, lse] = attention_run(q, k, v, mask, causal, scale, true);
    ctx->save_for_backward({q, k, v, mask, out, lse});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["D"] = q_in.size(3);
    // A narrower result is a copy: autograd would not see `out` change with a view of it made here.
    return out.size(3) == q_in.size(3) ? out : head_cols(out, q_in.size(3)).clone();
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(7);
    auto s = ctx->get_saved_variables();
    c10::OptionalDeviceGuard guard(s[0].device());
    auto [dq, dk, dv] = attention_grads(grads[0], s[0], s[1], s[2], s[3], s[4], s[5],
                                        ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble());
    const int64_t D = ctx->saved_data["D"].toInt();
    return once({head_cols(dq, D), head_cols(dk, D), head_cols(dv, D), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor attention_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const c10::optional<Tensor>& mask,
                          bool causal, double scale) {
  return AttentionFn::apply(q, k, v, mask.has_value() ? *mask : q, mask.has_value(), causal, scale);
}
Tensor attention_cuda(const Tensor& q, const Tensor& k, const Tensor& v, const c10::optional<Tensor>& mask,
                      bool causal, double scale) {
  c10::OptionalDeviceGuard guard(q.device());
  return head_cols(std::get<0>(attention_run(attention_rows(q), attention_rows(k), attention_rows(v),
                                             attention_mask(mask), causal, scale, false)),
                   q.size(3));
}

// ---- LayerNorm ----------------------------------------------------------------------------

struct NormOut {
  Tensor y, mean, rstd;
};

NormOut norm_run(const Tensor& x, const Tensor& r, const Tensor& w, const Tensor& b, double eps, bool with_stats) {
  const int64_t D = x.size(-1), M = D == 0 ? 0 : x.numel() / D;
  NormOut o;
  o.y = at::empty(x.sizes(), x.options());
  if (with_stats) {
    o.mean = at::empty({M}, x.options().dtype(at::kFloat));
    o.rstd = at::empty_like(o.mean);
  }
  check(sparton_layer_norm_fwd(x.data_ptr(), ptr(r), w.data_ptr(), ptr(b), dtype_code(w.scalar_type()), (float)eps,
                               o.y.data_ptr(), with_stats ? o.mean.data_ptr<float>() : nullptr,
                               with_stats ? o.rstd.data_ptr<float>() : nullptr, M, D, dtype_code(x.scalar_type()),
                               stream_of(x)),
        "sparton_layer_norm_fwd");
  return o;
}

std::tuple<Tensor, Tensor, Tensor> norm_grads(const Tensor& dy_in, const Tensor& x, const Tensor& r, const Tensor& w,
                                              bool has_bias, const Tensor& mean, const Tensor& rstd) {
  const int64_t D = x.size(-1), M = mean.size(0);
  Tensor dy = dy_in.to(x.scalar_type()).contiguous();
  Tensor dx = at::empty(x.sizes(), x.options());
  Tensor dw = at::empty({D}, w.options());
  Tensor db = at::empty({has_bias ? D : 0}, w.options());
  const size_t ws_bytes = sparton_layer_norm_workspace_bytes(M, D);
  Tensor ws = workspace(ws_bytes, x);
  check(sparton_layer_norm_bwd(dy.data_ptr(), x.data_ptr(), ptr(r), w.data_ptr(), dtype_code(w.scalar_type()),
                               mean.data_ptr<float>(), rstd.data_ptr<float>(), dx.data_ptr(), dw.data_ptr(),
                               has_bias ? db.data_ptr() : nullptr, ws.data_ptr(), ws_bytes, M, D,
                               dtype_code(x.scalar_type()), stream_of(x)),
        "sparton_layer_norm_bwd");
  return {dx, dw, db};
}

Tensor whole(const c10::optional<Tensor>& t) { return t.has_value() ? t->contiguous() : Tensor(); }

std::tuple<Tensor, Tensor, Tensor> norm_fwd_cuda(const Tensor& x, const c10::optional<Tensor>& r, const Tensor& w,
                                                 const c10::optional<Tensor>& b, double eps) {
  c10::OptionalDeviceGuard guard(x.device());
  NormOut o = norm_run(x.contiguous(), whole(r), w.contiguous(), whole(b), eps, true);
  return {o.y, o.mean, o.rstd};
}
std::tuple<Tensor, Tensor, Tensor> norm_bwd_cuda(const Tensor& dy, const Tensor& x, const c10::optional<Tensor>& r,
                                                 const Tensor& w, bool has_bias, const Tensor& mean,
                                                 const Tensor& rstd) {
  c10::OptionalDeviceGuard guard(x.device());
  return norm_grads(dy, x.contiguous(), whole(r), w.contiguous(), has_bias, mean, rstd);
}

struct NormFn : public torch::autograd::Function<NormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& r_in, const Tensor& w_in,
                        const Tensor& b_in, bool has_r, bool has_b, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    c10::OptionalDeviceGuard guard(x_in.device());
    Tensor x = x_in.contiguous(), r = has_r ? r_in.contiguous() : Tensor(), w = w_in.contiguous();
    NormOut o = norm_run(x, r, w, has_b ? b_in.contiguous() : Tensor(), eps, true);
    ctx->save_for_backward({x, r, w, o.mean, o.rstd});
    ctx->saved_data["has_b"] = has_b;
    return o.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(7);
    auto s = ctx->get_saved_variables();
    c10::OptionalDeviceGuard guard(s[0].device());
    const bool has_b = ctx->saved_data["has_b"].toBool();
    auto [dx, dw, db] = norm_grads(grads[0], s[0], s[1], s[2], has_b, s[3], s[4]);
    return once({dx, s[1].defined() ? dx : Tensor(), dw, has_b ? db : Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor norm_autograd(const Tensor& x, const c10::optional<Tensor>& r, const Tensor& w, const c10::optional<Tensor>& b,
                     double eps) {
  return NormFn::apply(x, r.has_value() ? *r : x, w, b.has_value() ? *b : w, r.has_value(), b.has_value(), eps);
}
Tensor norm_cuda(const Tensor& x, const c10::optional<Tensor>& r, const Tensor& w, const c10::optional<Tensor>& b,
                 double eps) {
  c10::OptionalDeviceGuard guard(x.device());
  return norm_run(x.contiguous(), whole(r), w.contiguous(), whole(b), eps, false).y;
}

// ---- the preference loss -------------------------------------------------------------------

// loss (undefined without `with_loss`), margin [B] and the backward's coefficients [B].
std::tuple<Tensor, Tensor, Tensor> preference_run(const Tensor& q, const Tensor& p, const Tensor& n, const Tensor& ref,
                                                  double T, double beta, double smoothing, bool with_loss) {
  const int64_t B = q.size(0), V = q.size(1);
  const auto f32 = q.options().dtype(at::kFloat);
  Tensor margin = at::empty({B}, f32);
  Tensor loss = with_loss ? at::empty({}, f32) : Tensor(), coef = with_loss ? at::empty({B}, f32) : Tensor();
  const int dt = dtype_code(q.scalar_type());
  const size_t ws_bytes = sparton_preference_workspace_bytes(B, V, dt);
  Tensor ws = workspace(ws_bytes, q);
  check(sparton_preference_fwd(q.data_ptr(), p.data_ptr(), n.data_ptr(), ref.defined() ? ref.data_ptr<float>() : nullptr,
                               B, V, (float)T, (float)beta, (float)smoothing,
                               with_loss ? loss.data_ptr<float>() : nullptr, margin.data_ptr<float>(),
                               with_loss ? coef.data_ptr<float>() : nullptr, ws.data_ptr(), ws_bytes, dt, stream_of(q)),
        "sparton_preference_fwd");
  return {loss, margin, coef};
}

std::tuple<Tensor, Tensor, Tensor> preference_grads(const Tensor& grad, const Tensor& q, const Tensor& p,
                                                    const Tensor& n, const Tensor& coef) {
  Tensor g = grad.to(at::kFloat).contiguous();
  Tensor dq = at::empty(q.sizes(), q.options()), dp = at::empty_like(dq), dn = at::empty_like(dq);
  check(sparton_preference_bwd(q.data_ptr(), p.data_ptr(), n.data_ptr(), coef.data_ptr<float>(), g.data_ptr<float>(),
                               q.size(0), q.size(1), dq.data_ptr(), dp.data_ptr(), dn.data_ptr(),
                               dtype_code(q.scalar_type()), stream_of(q)),
        "sparton_preference_bwd");
  return {dq, dp, dn};
}

std::tuple<Tensor, Tensor, Tensor> preference_fwd_cuda(const Tensor& q, const Tensor& p, const Tensor& n,
                                                       const c10::optional<Tensor>& ref, double T, double beta,
                                                       double smoothing) {
  c10::OptionalDeviceGuard guard(q.device());
  return preference_run(q.contiguous(), p.contiguous(), n.contiguous(), whole(ref), T, beta, smoothing, true);
}
std::tuple<Tensor, Tensor, Tensor> preference_bwd_cuda(const Tensor& grad, const Tensor& q, const Tensor& p,
                                                       const Tensor& n, const Tensor& coef) {
  c10::OptionalDeviceGuard guard(q.device());
  return preference_grads(grad, q.contiguous(), p.contiguous(), n.contiguous(), coef);
}
Tensor preference_margin_cuda(const Tensor& q, const Tensor& p, const Tensor& n, double T) {
  c10::OptionalDeviceGuard guard(q.device());
  return std::get<1>(preference_run(q.contiguous(), p.contiguous(), n.contiguous(), Tensor(), T, 1.0, 0.0, false));
}

struct PreferenceFn : public torch::autograd::Function<PreferenceFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q_in, const Tensor& p_in, const Tensor& n_in,
                               const Tensor& ref, bool has_ref, double T, double beta, double smoothing) {
    at::AutoDispatchBelowADInplaceOrView below;
    c10::OptionalDeviceGuard guard(q_in.device());
    Tensor q = q_in.contiguous(), p = p_in.contiguous(), n = n_in.contiguous();
    auto [loss, margin, coef] = preference_run(q, p, n, has_ref ? ref.contiguous() : Tensor(), T, beta, smoothing, true);
    ctx->save_for_backward({q, p, n, coef});
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({margin});
    return {loss, margin};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(8);
    auto s = ctx->get_saved_variables();
    c10::OptionalDeviceGuard guard(s[0].device());
    auto [dq, dp, dn] = preference_grads(grads[0], s[0], s[1], s[2], s[3]);
    return once({dq, dp, dn, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

std::tuple<Tensor, Tensor> preference_autograd(const Tensor& q, const Tensor& p, const Tensor& n,
                                               const c10::optional<Tensor>& ref, double T, double beta,
                                               double smoothing) {
  auto o = PreferenceFn::apply(q, p, n, ref.has_value() ? *ref : q, ref.has_value(), T, beta, smoothing);
  return {o[0], o[1]};
}
std::tuple<Tensor, Tensor> preference_cuda(const Tensor& q, const Tensor& p, const Tensor& n,
                                           const c10::optional<Tensor>& ref, double T, double beta, double smoothing) {
  auto [loss, margin, coef] = preference_fwd_cuda(q, p, n, ref, T, beta, smoothing);
  return {loss, margin};
}

// Whether a graph is to be kept: the dispatcher calls the autograd kernels without one too.
template <typename... T> bool wants_grad(const T&... t) {
  return at::GradMode::is_enabled() && ((t.defined() && t.requires_grad()) || ...);
}

// A forward-mode derivative rides on a tensor that asks for no gradient; without a graph node to refuse it, it would
// be lost.
template <typename... T> void refuse_forward_mode(const char* what, const T&... t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!((t.defined() && t._fw_grad(0).defined()) || ...), "sparton: ", what,
                              " has no forward-mode derivative");
}

// ---- the RMS norm --------------------------------------------------------------------------

struct RmsOut {
  Tensor y, h, rstd;
};

RmsOut rms_run(const Tensor& x, const Tensor& r, const Tensor& w, double eps, bool with_stats) {
  const int64_t D = x.size(-1), M = D == 0 ? 0 : x.numel() / D;
  RmsOut o;
  o.y = at::empty(x.sizes(), x.options());
  if (r.defined()) o.h = at::empty(x.sizes(), x.options());
  if (with_stats) o.rstd = at::empty({M}, x.options().dtype(at::kFloat));
  check(sparton_rms_norm_fwd(x.data_ptr(), ptr(r), w.data_ptr(), dtype_code(w.scalar_type()), (float)eps, o.y.data_ptr(),
                             mptr(o.h), with_stats ? o.rstd.data_ptr<float>() : nullptr, M, D, dtype_code(x.scalar_type()),
                             stream_of(x)),
        "sparton_rms_norm_fwd");
  return o;
}

std::tuple<Tensor, Tensor> rms_grads(const Tensor& dy_in, const Tensor& dh_in, const Tensor& h, const Tensor& w,
                                     const Tensor& rstd, bool with_dw) {
  const int64_t D = h.size(-1), M = rstd.size(0);
  Tensor dy = dy_in.to(h.scalar_type()).contiguous();
  Tensor dh = dh_in.defined() ? dh_in.to(h.scalar_type()).contiguous() : Tensor();
  Tensor dx = at::empty(h.sizes(), h.options());
  Tensor dw = with_dw ? at::empty({D}, w.options()) : Tensor();
  const size_t ws_bytes = sparton_rms_norm_workspace_bytes(M, D);
  Tensor ws = workspace(ws_bytes, h);
  check(sparton_rms_norm_bwd(dy.data_ptr(), ptr(dh), h.data_ptr(), w.data_ptr(), dtype_code(w.scalar_type()),
                             rstd.data_ptr<float>(), dx.data_ptr(), mptr(dw), ws.data_ptr(), ws_bytes, M, D,
                             dtype_code(h.scalar_type()), stream_of(h)),
        "sparton_rms_norm_bwd");
  return {dx, dw};
}

std::tuple<Tensor, Tensor, Tensor> rms_fwd_cuda(const Tensor& x, const c10::optional<Tensor>& r, const Tensor& w, double eps) {
  c10::OptionalDeviceGuard guard(x.device());
  RmsOut o = rms_run(x.contiguous(), whole(r), w.contiguous(), eps, true);
  return {o.y, o.h.defined() ? o.h : at::empty({0}, x.options()), o.rstd};
}
std::tuple<Tensor, Tensor> rms_bwd_cuda(const Tensor& dy, const c10::optional<Tensor>& dh, const Tensor& h, const Tensor& w,
                                        const Tensor& rstd) {
  c10::OptionalDeviceGuard guard(h.device());
  return rms_grads(dy, whole(dh), h.contiguous(), w.contiguous(), rstd, true);
}

struct RmsFn : public torch::autograd::Function<RmsFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& r_in, const Tensor& w_in, bool has_r,
                               double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    c10::OptionalDeviceGuard guard(x_in.device());
    Tensor x = x_in.contiguous(), w = w_in.contiguous();
    RmsOut o = rms_run(x, has_r ? r_in.contiguous() : Tensor(), w, eps, true);
    ctx->save_for_backward({has_r ? o.h : x, w, o.rstd});
    ctx->saved_data["has_r"] = has_r;
    ctx->set_materialize_grads(false);
    return has_r ? variable_list{o.y, o.h} : variable_list{o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool has_r = ctx->saved_data["has_r"].toBool();
    const Tensor dh = has_r ? grads[1] : Tensor();
    if (!grads[0].defined()) return once({dh, dh, Tensor(), Tensor(), Tensor()});
    auto s = ctx->get_saved_variables();
    c10::OptionalDeviceGuard guard(s[0].device());
    auto [dx, dw] = rms_grads(grads[0], dh, s[0], s[1], s[2], ctx->needs_input_grad(2));
    return once({dx, has_r ? dx : Tensor(), dw, Tensor(), Tensor()});
  }
};

Tensor rms_cuda(const Tensor& x, const Tensor& w, double eps) {
  c10::OptionalDeviceGuard guard(x.device());
  return rms_run(x.contiguous(), Tensor(), w.contiguous(), eps, false).y;
}
std::tuple<Tensor, Tensor> rms_add_cuda(const Tensor& x, const Tensor& r, const Tensor& w, double eps) {
  c10::OptionalDeviceGuard guard(x.device());
  RmsOut o = rms_run(x.contiguous(), r.contiguous(), w.contiguous(), eps, false);
  return {o.y, o.h};
}
Tensor rms_autograd(const Tensor& x, const Tensor& w, double eps) {
  refuse_forward_mode("rms_norm", x, w);
  if (wants_grad(x, w)) return RmsFn::apply(x, x, w, false, eps)[0];
  at::AutoDispatchBelowADInplaceOrView below;
  return rms_cuda(x, w, eps);
}
std::tuple<Tensor, Tensor> rms_add_autograd(const Tensor& x, const Tensor& r, const Tensor& w, double eps) {
  refuse_forward_mode("rms_norm", x, r, w);
  if (wants_grad(x, r, w)) {
    auto o = RmsFn::apply(x, r, w, true, eps);
    return {o[0], o[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return rms_add_cuda(x, r, w, eps);
}
std::tuple<Tensor, Tensor, Tensor> rms_8bit_cuda(const Tensor& x_in, const c10::optional<Tensor>& r_in, const Tensor& w_in,
                                                 double eps) {
  c10::OptionalDeviceGuard guard(x_in.device());
  Tensor x = x_in.contiguous(), r = whole(r_in), w = w_in.contiguous();
  const int64_t D = x.size(-1), M = D == 0 ? 0 : x.numel() / D;
  Tensor y = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
  Tensor scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  Tensor h = r.defined() ? at::empty(x.sizes(), x.options()) : at::empty({0}, x.options());
  check(sparton_rms_norm_fwd_quantized(x.data_ptr(), ptr(r), w.data_ptr(), dtype_code(w.scalar_type()), (float)eps, y.data_ptr(),
                                  scale.data_ptr<float>(), r.defined() ? h.data_ptr() : nullptr, M, D,
                                  dtype_code(x.scalar_type()), stream_of(x)),
        "sparton_rms_norm_fwd_quantized");
  return {y, scale, h};
}
std::tuple<Tensor, Tensor, Tensor> rms_8bit_autograd(const Tensor& x, const c10::optional<Tensor>& r, const Tensor& w, double eps) {
  refuse_forward_mode("rms_norm_8bit", x, opt(r), w);
  at::AutoDispatchBelowADInplaceOrView below;
  return rms_8bit_cuda(x, r, w, eps);
}

// ---- the embedding -------------------------------------------------------------------------

Tensor embedding_run(const Tensor& ids, const Tensor& w, double scale) {
  auto shape = ids.sizes().vec();
  shape.push_back(w.size(1));
  Tensor out = at::empty(shape, w.options());
  check(sparton_embedding_fwd(ids.data_ptr(), mask_code(ids.scalar_type()), w.data_ptr(), (float)scale, out.data_ptr(),
                              ids.numel(), w.size(0), w.size(1), dtype_code(w.scalar_type()), stream_of(w)),
        "sparton_embedding_fwd");
  return out;
}

Tensor embedding_grad(const Tensor& d_out, const Tensor& ids, int64_t rows, double scale, int64_t padding) {
  Tensor g = d_out.contiguous();
  const int64_t N = ids.numel(), D = g.size(-1);
  Tensor dw = at::empty({rows, D}, g.options());
  const int dt = dtype_code(g.scalar_type());
  const size_t ws_bytes = sparton_embedding_workspace_bytes(N, rows, D, dt);
  Tensor ws = workspace(ws_bytes, g);
  check(sparton_embedding_bwd(ids.data_ptr(), mask_code(ids.scalar_type()), g.data_ptr(), (float)scale, padding, dw.data_ptr(),
                              ws.data_ptr(), ws_bytes, N, rows, D, dt, stream_of(g)),
        "sparton_embedding_bwd");
  return dw;
}

Tensor embedding_cuda(const Tensor& ids, const Tensor& w, double scale, int64_t) {
  c10::OptionalDeviceGuard guard(w.device());
  return embedding_run(ids.contiguous(), w.contiguous(), scale);
}
Tensor embedding_bwd_cuda(const Tensor& d_out, const Tensor& ids, int64_t rows, double scale, int64_t padding) {
  c10::OptionalDeviceGuard guard(d_out.device());
  return embedding_grad(d_out, ids.contiguous(), rows, scale, padding);
}

struct EmbeddingFn : public torch::autograd::Function<EmbeddingFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids_in, const Tensor& w, double scale, int64_t padding) {
    at::AutoDispatchBelowADInplaceOrView below;
    c10::OptionalDeviceGuard guard(w.device());
    Tensor ids = ids_in.contiguous();
    const int64_t N = ids.numel(), V = w.size(0), D = w.size(1);
    TORCH_CHECK(N == 0 || V == 0 || sparton_embedding_workspace_bytes(N, V, D, dtype_code(w.scalar_type())) > 0,
                "sparton: embedding: ", N, " ids of rows of ", D, " are too many for a gradient");
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = w.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    ctx->saved_data["dtype"] = (int64_t)w.scalar_type();
    return embedding_run(ids, w.contiguous(), scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(4);
    auto s = ctx->get_saved_variables();
    c10::OptionalDeviceGuard guard(s[0].device());
    Tensor g = grads[0].to((at::ScalarType)ctx->saved_data["dtype"].toInt());
    return once({Tensor(), embedding_grad(g, s[0], ctx->saved_data["rows"].toInt(), ctx->saved_data["scale"].toDouble(),
                                          ctx->saved_data["padding"].toInt()),
                 Tensor(), Tensor()});
  }
};

Tensor embedding_autograd(const Tensor& ids, const Tensor& w, double scale, int64_t padding) {
  refuse_forward_mode("embedding", w);
  if (wants_grad(w)) return EmbeddingFn::apply(ids, w, scale, padding);
  at::AutoDispatchBelowADInplaceOrView below;
  return embedding_cuda(ids, w, scale, padding);
}

// ---- the gated feed-forward product --------------------------------------------------------

// Rows of whole 16 bytes, as the C ABI reads them: a width that is not is padded with zero columns, which change
// no product.
Tensor gated_rows(const Tensor& t) {
  const int64_t unit = 16 / t.element_size(), pad = (unit - t.size(-1) % unit) % unit;
  return pad > 0 ? at::constant_pad_nd(t.element_size() == 1 ? t.view(at::kByte) : t, {0, pad}).contiguous() : dense(t);
}

struct GatedOut {
  Tensor h, g, u;
};

// x [..., D] and the weights [F, D] as gated_rows gives them.
GatedOut gated_run(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& bg, const Tensor& bu, int64_t act,
                   bool with_saved) {
  const int64_t D = x.size(-1), F = wg.size(0), M = x.numel() / D;
  auto shape = x.sizes().vec();
  shape.back() = F;
  GatedOut o;
  o.h = at::empty(shape, x.options());
  if (with_saved) {
    o.g = at::empty({M, F}, x.options().dtype(at::kFloat));
    o.u = at::empty_like(o.g);
  }
  check(sparton_gated_fwd(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), ptr(bg), ptr(bu), (int)act, o.h.data_ptr(),
                          with_saved ? o.g.data_ptr<float>() : nullptr, with_saved ? o.u.data_ptr<float>() : nullptr, M, D, F,
                          dtype_code(x.scalar_type()), stream_of(x)),
        "sparton_gated_fwd");
  return o;
}

// (dx, dw_gate, dw_up, db_gate, db_up) of width D; what is not asked for stays undefined.
variable_list gated_grads(const Tensor& dh_in, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& g,
                          const Tensor& u, int64_t act, int64_t D, bool need_x, bool need_w, bool need_bg, bool need_bu) {
  const int64_t P = x.size(-1), F = wg.size(0), M = g.size(0);
  Tensor dh = dh_in.to(x.scalar_type()).contiguous();
  variable_list d(5);
  if (need_x) d[0] = at::empty(x.sizes(), x.options());
  if (need_w) d[1] = at::empty(wg.sizes(), x.options()), d[2] = at::empty_like(d[1]);
  if (need_bg) d[3] = at::empty({F}, x.options());
  if (need_bu) d[4] = at::empty({F}, x.options());
  const int dt = dtype_code(x.scalar_type());
  if (F == 0) {
    for (Tensor& t : d)
      if (t.defined()) t.zero_();
  } else {
    const size_t ws_bytes = sparton_gated_workspace_bytes(M, P, F, need_bg || need_bu, dt);
    Tensor ws = workspace(ws_bytes, x);
    check(sparton_gated_bwd(dh.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), g.data_ptr<float>(), u.data_ptr<float>(),
                            (int)act, mptr(d[0]), mptr(d[1]), mptr(d[2]), mptr(d[3]), mptr(d[4]), ws.data_ptr(), ws_bytes, M, P, F,
                            dt, stream_of(x)),
          "sparton_gated_bwd");
  }
  for (int i = 0; i < 3; ++i)
    if (d[i].defined() && P != D) d[i] = d[i].narrow(-1, 0, D).contiguous();
  return d;
}

std::tuple<Tensor, Tensor, Tensor> gated_fwd_cuda(const Tensor& x, const Tensor& wg, const Tensor& wu,
                                                  const c10::optional<Tensor>& bg, const c10::optional<Tensor>& bu, int64_t act) {
  c10::OptionalDeviceGuard guard(x.device());
  GatedOut o = gated_run(gated_rows(x), gated_rows(wg), gated_rows(wu), whole(bg), whole(bu), act, true);
  return {o.h, o.g, o.u};
}
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> gated_bwd_cuda(const Tensor& dh, const Tensor& x, const Tensor& wg,
                                                                  const Tensor& wu, const Tensor& g, const Tensor& u,
                                                                  int64_t act, bool has_bg, bool has_bu, bool need_x,
                                                                  bool need_w) {
  c10::OptionalDeviceGuard guard(x.device());
  auto d = gated_grads(dh, gated_rows(x), gated_rows(wg), gated_rows(wu), g, u, act, x.size(-1), need_x, need_w, has_bg, has_bu);
  for (Tensor& t : d)
    if (!t.defined()) t = at::empty({0}, x.options());
  return {d[0], d[1], d[2], d[3], d[4]};
}

struct GatedFn : public torch::autograd::Function<GatedFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& wg_in, const Tensor& wu_in, const Tensor& bg,
                        const Tensor& bu, bool has_bg, bool has_bu, int64_t act) {
    at::AutoDispatchBelowADInplaceOrView below;
    c10::OptionalDeviceGuard guard(x_in.device());
    Tensor x = gated_rows(x_in), wg = gated_rows(wg_in), wu = gated_rows(wu_in);
    GatedOut o = gated_run(x, wg, wu, has_bg ? bg.contiguous() : Tensor(), has_bu ? bu.contiguous() : Tensor(), act, true);
    ctx->save_for_backward({x, wg, wu, o.g, o.u});
    ctx->saved_data["act"] = act;
    ctx->saved_data["D"] = x_in.size(-1);
    ctx->saved_data["has_bg"] = has_bg;
    ctx->saved_data["has_bu"] = has_bu;
    return o.h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(8);
    auto s = ctx->get_saved_variables();
    c10::OptionalDeviceGuard guard(s[0].device());
    const auto need = [&](size_t i) { return ctx->needs_input_grad(i); };
    auto d = gated_grads(grads[0], s[0], s[1], s[2], s[3], s[4], ctx->saved_data["act"].toInt(), ctx->saved_data["D"].toInt(),
                         need(0), need(1) || need(2), ctx->saved_data["has_bg"].toBool() && need(3),
                         ctx->saved_data["has_bu"].toBool() && need(4));
    return once({d[0], d[1], d[2], d[3], d[4], Tensor(), Tensor(), Tensor()});
  }
};

Tensor gated_cuda(const Tensor& x, const Tensor& wg, const Tensor& wu, const c10::optional<Tensor>& bg,
                  const c10::optional<Tensor>& bu, int64_t act) {
  c10::OptionalDeviceGuard guard(x.device());
  return gated_run(gated_rows(x), gated_rows(wg), gated_rows(wu), whole(bg), whole(bu), act, false).h;
}
Tensor gated_autograd(const Tensor& x, const Tensor& wg, const Tensor& wu, const c10::optional<Tensor>& bg,
                      const c10::optional<Tensor>& bu, int64_t act) {
  refuse_forward_mode("gated_linear", x, wg, wu, opt(bg), opt(bu));
  if (wants_grad(x, wg, wu, bg.value_or(Tensor()), bu.value_or(Tensor())))
    return GatedFn::apply(x, wg, wu, bg.has_value() ? *bg : x, bu.has_value() ? *bu : x, bg.has_value(), bu.has_value(), act);
  at::AutoDispatchBelowADInplaceOrView below;
  return gated_cuda(x, wg, wu, bg, bu, act);
}
Tensor gated_8bit_cuda(const Tensor& x_in, const Tensor& sx, const Tensor& wg_in, const Tensor& sg, const Tensor& wu_in,
                       const Tensor& su, int64_t act, at::ScalarType out_dtype) {
  c10::OptionalDeviceGuard guard(x_in.device());
  Tensor x = gated_rows(x_in), wg = gated_rows(wg_in), wu = gated_rows(wu_in);
  const int64_t D = x.size(-1), F = wg.size(0), M = x.numel() / D;
  auto shape = x.sizes().vec();
  shape.back() = F;
  Tensor h = at::empty(shape, x.options().dtype(out_dtype));
  Tensor a = sx.contiguous(), b = sg.contiguous(), c = su.contiguous();
  check(sparton_gated_fwd_quantized(x.data_ptr(), a.data_ptr<float>(), wg.data_ptr(), b.data_ptr<float>(), wu.data_ptr(),
                               c.data_ptr<float>(), (int)act, h.data_ptr(), M, D, F, dtype_code(out_dtype), stream_of(x)),
        "sparton_gated_fwd_quantized");
  return h;
}
Tensor gated_8bit_autograd(const Tensor& x, const Tensor& sx, const Tensor& wg, const Tensor& sg, const Tensor& wu,
                           const Tensor& su, int64_t act, at::ScalarType out_dtype) {
  refuse_forward_mode("gated_linear_8bit", x, sx, wg, sg, wu, su);
  at::AutoDispatchBelowADInplaceOrView below;
  return gated_8bit_cuda(x, sx, wg, sg, wu, su, act, out_dtype);
}

// CPU tensors: the same refusal as the reference's `assert hidden.is_cuda`
// (sparton_kernel.py:650), as a RuntimeError.
[[noreturn]] void cpu_refused(const char* op) {
  TORCH_CHECK(false, op, " only supports ROCm/HIP device tensors (got a CPU tensor)");
}

}  // namespace

TORCH_LIBRARY(sparton_eager, m) {
  m.def("head_train(Tensor hidden, Tensor weight, Tensor? bias, Tensor mask) -> Tensor");
  m.def("head_encode(Tensor hidden, Tensor weight, Tensor? bias, Tensor mask) -> Tensor");
  m.def("head_train_autocast(Tensor hidden, Tensor weight, Tensor? bias, Tensor mask, "
        "Tensor weight_c, Tensor? bias_c, int pad) -> Tensor");
  m.def("mlm_transform(Tensor x, Tensor weight, Tensor dense_bias, Tensor ln_weight, "
        "Tensor ln_bias, float eps) -> Tensor");
  m.def("mlm_transform_typed(Tensor x, Tensor weight, Tensor dense_bias, Tensor ln_weight, "
        "Tensor ln_bias, float eps) -> Tensor");
  m.def("splade_loss(Tensor q, Tensor? d, float temperature, float w_ce, float w_l1, "
        "float w_flops) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("attention(Tensor q, Tensor k, Tensor v, Tensor? mask, bool causal, float scale) -> Tensor");
  m.def("attention_fwd(Tensor q, Tensor k, Tensor v, Tensor? mask, bool causal, float scale) -> (Tensor, Tensor)");
  m.def("attention_bwd(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor? mask, Tensor out, Tensor lse, "
        "bool causal, float scale) -> (Tensor, Tensor, Tensor)");
  m.def("layer_norm(Tensor x, Tensor? residual, Tensor weight, Tensor? bias, float eps) -> Tensor");
  m.def("layer_norm_fwd(Tensor x, Tensor? residual, Tensor weight, Tensor? bias, float eps) "
        "-> (Tensor, Tensor, Tensor)");
  m.def("layer_norm_bwd(Tensor dy, Tensor x, Tensor? residual, Tensor weight, bool has_bias, Tensor mean, "
        "Tensor rstd) -> (Tensor, Tensor, Tensor)");
  m.def("preference_loss(Tensor q, Tensor pos, Tensor neg, Tensor? ref_margin, float temperature, float beta, "
        "float smoothing) -> (Tensor, Tensor)");
  m.def("preference_fwd(Tensor q, Tensor pos, Tensor neg, Tensor? ref_margin, float temperature, float beta, "
        "float smoothing) -> (Tensor, Tensor, Tensor)");
  m.def("preference_bwd(Tensor grad, Tensor q, Tensor pos, Tensor neg, Tensor coef) -> (Tensor, Tensor, Tensor)");
  m.def("preference_margin(Tensor q, Tensor pos, Tensor neg, float temperature) -> Tensor");
  m.def("rms_norm(Tensor x, Tensor weight, float eps) -> Tensor");
  m.def("rms_norm_add(Tensor x, Tensor residual, Tensor weight, float eps) -> (Tensor, Tensor)");
  m.def("rms_norm_fwd(Tensor x, Tensor? residual, Tensor weight, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("rms_norm_bwd(Tensor dy, Tensor? dh, Tensor h, Tensor weight, Tensor rstd) -> (Tensor, Tensor)");
  m.def("rms_norm_8bit(Tensor x, Tensor? residual, Tensor weight, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("embedding(Tensor ids, Tensor weight, float scale, int padding) -> Tensor");
  m.def("embedding_bwd(Tensor d_out, Tensor ids, int rows, float scale, int padding) -> Tensor");
  m.def("gated(Tensor x, Tensor w_gate, Tensor w_up, Tensor? b_gate, Tensor? b_up, int activation) -> Tensor");
  m.def("gated_fwd(Tensor x, Tensor w_gate, Tensor w_up, Tensor? b_gate, Tensor? b_up, int activation) "
        "-> (Tensor, Tensor, Tensor)");
  m.def("gated_bwd(Tensor dh, Tensor x, Tensor w_gate, Tensor w_up, Tensor gate, Tensor up, int activation, "
        "bool has_b_gate, bool has_b_up, bool need_x=True, bool need_w=True) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("gated_8bit(Tensor x, Tensor x_scale, Tensor w_gate, Tensor gate_scale, Tensor w_up, Tensor up_scale, "
        "int activation, ScalarType out_dtype) -> Tensor");
}

TORCH_LIBRARY_IMPL(sparton_eager, CUDA, m) {
  m.impl("head_train", &head_train_cuda);
  m.impl("head_encode", &head_encode_cuda);
  m.impl("head_train_autocast", &head_train_autocast_cuda);
  m.impl("mlm_transform", &transform_cuda);
  m.impl("mlm_transform_typed", &transform_typed_cuda);
  m.impl("splade_loss", &loss_cuda);
  m.impl("attention", &attention_cuda);
  m.impl("attention_fwd", &attention_fwd_cuda);
  m.impl("attention_bwd", &attention_bwd_cuda);
  m.impl("layer_norm", &norm_cuda);
  m.impl("layer_norm_fwd", &norm_fwd_cuda);
  m.impl("layer_norm_bwd", &norm_bwd_cuda);
  m.impl("preference_loss", &preference_cuda);
  m.impl("preference_fwd", &preference_fwd_cuda);
  m.impl("preference_bwd", &preference_bwd_cuda);
  m.impl("preference_margin", &preference_margin_cuda);
  m.impl("rms_norm", &rms_cuda);
  m.impl("rms_norm_add", &rms_add_cuda);
  m.impl("rms_norm_fwd", &rms_fwd_cuda);
  m.impl("rms_norm_bwd", &rms_bwd_cuda);
  m.impl("rms_norm_8bit", &rms_8bit_cuda);
  m.impl("embedding", &embedding_cuda);
  m.impl("embedding_bwd", &embedding_bwd_cuda);
  m.impl("gated", &gated_cuda);
  m.impl("gated_fwd", &gated_fwd_cuda);
  m.impl("gated_bwd", &gated_bwd_cuda);
  m.impl("gated_8bit", &gated_8bit_cuda);
}

TORCH_LIBRARY_IMPL(sparton_eager, AutogradCUDA, m) {
  m.impl("head_train", &head_train_autograd);
  m.impl("head_train_autocast", &head_train_autocast_autograd);
  m.impl("mlm_transform", &transform_autograd);
  m.impl("mlm_transform_typed", &transform_typed_autograd);
  m.impl("splade_loss", &loss_autograd);
  m.impl("attention", &attention_autograd);
  m.impl("layer_norm", &norm_autograd);
  m.impl("preference_loss", &preference_autograd);
  m.impl("rms_norm", &rms_autograd);
  m.impl("rms_norm_add", &rms_add_autograd);
  m.impl("rms_norm_8bit", &rms_8bit_autograd);
  m.impl("embedding", &embedding_autograd);
  m.impl("gated", &gated_autograd);
  m.impl("gated_8bit", &gated_8bit_autograd);
}

TORCH_LIBRARY_IMPL(sparton_eager, CPU, m) {
  m.impl("head_train", [](const Tensor&, const Tensor&, const c10::optional<Tensor>&, const Tensor&) -> Tensor {
    cpu_refused("sparton_eager::head_train");
  });
  m.impl("head_encode", [](const Tensor&, const Tensor&, const c10::optional<Tensor>&, const Tensor&) -> Tensor {
    cpu_refused("sparton_eager::head_encode");
  });
  m.impl("head_train_autocast",
         [](const Tensor&, const Tensor&, const c10::optional<Tensor>&, const Tensor&, const Tensor&,
            const c10::optional<Tensor>&, int64_t) -> Tensor { cpu_refused("sparton_eager::head_train_autocast"); });
  m.impl("mlm_transform", [](const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                             double) -> Tensor { cpu_refused("sparton_eager::mlm_transform"); });
  m.impl("mlm_transform_typed", [](const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                   double) -> Tensor { cpu_refused("sparton_eager::mlm_transform_typed"); });
  m.impl("splade_loss", [](const Tensor&, const c10::optional<Tensor>&, double, double, double,
                           double) -> Loss6 { cpu_refused("sparton_eager::splade_loss"); });
  m.impl("attention", [](const Tensor&, const Tensor&, const Tensor&, const c10::optional<Tensor>&, bool,
                         double) -> Tensor { cpu_refused("sparton_eager::attention"); });
  m.impl("layer_norm", [](const Tensor&, const c10::optional<Tensor>&, const Tensor&, const c10::optional<Tensor>&,
                          double) -> Tensor { cpu_refused("sparton_eager::layer_norm"); });
  m.impl("preference_loss", [](const Tensor&, const Tensor&, const Tensor&, const c10::optional<Tensor>&, double, double,
                               double) -> std::tuple<Tensor, Tensor> { cpu_refused("sparton_eager::preference_loss"); });
}
