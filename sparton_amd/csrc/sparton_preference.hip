// Preference loss on pairs of documents, forward and backward, on gfx950. A retriever gives document
// d the probability softmax over its scores q . d / T, so a pair's log ratio is its score margin:
//     m_i = (q_i . p_i - q_i . n_i) / T,   z_i = beta (m_i - r_i)   (r: the reference model's margins)
//     loss = mean_i [ -(1 - eps) log sigma(z_i) - eps log sigma(-z_i) ]
//     c_i = (sigma(z_i) - (1 - eps)) beta / (B T);   dq_i = c_i (p_i - n_i), dp_i = c_i q_i, dn_i = -c_i q_i
// Both passes are bound by memory. Forward: each workgroup sums one chunk of one row's q (p - n) (the
// difference first: two close scores would cancel), and one workgroup adds the chunks in order and
// forms margins, loss and c. Backward: one pass over the rows. At 500 rows of 250002 in bf16 the margins
// take 164 us (4.6 TB/s; a copy reaches 4.9), the one workgroup 5.6, and the gradients 257 (5.8); at 32 rows
// of 30522, 3.4, 2.2 and 4.2 us, mostly launches.
// Rows of V elements need no alignment (V = 30522 in 16 bits: rows start on 4 bytes): global vector
// accesses take any address, and a row's last vector is moved back to end with the row.

#include <math.h>

#include <algorithm>

#include "sparton_common.h"

namespace sparton {
namespace pref {

constexpr int NT = 256;
constexpr int FIN = 1024;             // threads of the finishing workgroup
constexpr int kMaxChunks = 64;
constexpr int64_t kMaxParts = 8192;
// A launch holds fewer than 2^32 threads (past that, workgroups were left out without an error), and a
// row takes at least one workgroup.
constexpr int64_t kMaxGroups = (((int64_t)1 << 32) - 1) / NT;

template <typename T> struct Vec {
  static constexpr int N = 16 / sizeof(T);
  typedef __attribute__((ext_vector_type(16 / sizeof(T)))) T type;
  typedef type loose __attribute__((aligned(sizeof(T))));
};
template <typename T> __device__ __forceinline__ typename Vec<T>::type load_any(const T* p) {
  return *(const typename Vec<T>::loose*)p;
}
template <typename T> __device__ __forceinline__ void store_any(T* p, typename Vec<T>::type v) {
  *(typename Vec<T>::loose*)p = v;
}

struct Plan {
  int64_t chunks;  // of a row, at most `cap`
  int64_t span;    // elements of a chunk, a multiple of a workgroup's step
};
Plan plan(int64_t V, int es, int64_t cap) {
  const int64_t step = NT * (16 / es);
  Plan p;
  p.span = std::max(2 * step, round_up(cdiv(V, cap), step));
  p.chunks = cdiv(V, p.span);
  return p;
}
// Short chunks in the rows' order keep the memory's open pages few: at 500 rows of 250002 in 16 bits
// margins took 157 us by 2 steps a chunk, 160 by 4, 164 by 8, 176 by 25; gradients 273, 256, 258 us by
// 1, 2, 4 steps and 302 by 25. One workgroup adds the margins' chunks (5 of a row
// in 4.8 us, 16 in 5.6, 31 in 7), so there they are limited.
Plan margin_plan(int64_t B, int64_t V, int es) {
  return plan(V, es, std::min<int64_t>(kMaxChunks, std::max<int64_t>(1, kMaxParts / B)));
}
Plan grad_plan(int64_t B, int64_t V, int es) { return plan(V, es, kMaxGroups / B); }

// Sum over the workgroup in a fixed order; result in thread 0.
template <int THREADS> __device__ __forceinline__ float group_sum(float x, float* lds) {
  x = wave_sum(x);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) s += lds[w];
  return s;
}

// Rows shorter than a vector (V < N) are read element by element.
template <typename T>
__global__ __launch_bounds__(NT) void pref_margin_kernel(const T* __restrict__ q, const T* __restrict__ p,
                                                         const T* __restrict__ n, int64_t V, int64_t chunks, int64_t span,
                                                         float* __restrict__ part) {
  constexpr int N = Vec<T>::N;
  __shared__ float lds[NT / 64];
  const int64_t b = blockIdx.x / chunks, v0 = (int64_t)(blockIdx.x % chunks) * span, v1 = min(V, v0 + span);
  const int64_t base = b * V;
  float a = 0.0f;
  if (V >= N) {
#pragma unroll 4
    for (int64_t v = v0 + threadIdx.x * N; v < v1; v += NT * N) {
      const int64_t at = min(v, V - N);
      const int own = (int)(v - at);
      const auto qv = load_any<T>(q + base + at), pv = load_any<T>(p + base + at), nv = load_any<T>(n + base + at);
#pragma unroll
      for (int e = 0; e < N; ++e) a += e >= own ? to_f32(qv[e]) * (to_f32(pv[e]) - to_f32(nv[e])) : 0.0f;
    }
  } else if ((int64_t)threadIdx.x < V) {
    const int64_t at = base + threadIdx.x;
    a = to_f32(q[at]) * (to_f32(p[at]) - to_f32(n[at]));
  }
  a = group_sum<NT>(a, lds);
  if (threadIdx.x == 0) part[blockIdx.x] = a;
}

// log(1 + exp(-|z|)) and sigma(|z|)'s complement, without overflow.
__device__ __forceinline__ float softplus_tail(float z) { return log1p_pos(__builtin_amdgcn_exp2f(-fabsf(z) * 1.44269504088896341f)); }

__global__ __launch_bounds__(FIN) void pref_finish_kernel(const float* __restrict__ part, int chunks,
                                                          const float* __restrict__ ref, int64_t B, float inv_t,
                                                          float beta, float smoothing, float* __restrict__ loss,
                                                          float* __restrict__ margin, float* __restrict__ coef) {
  __shared__ float lds[FIN / 64];
  float total = 0.0f;
  for (int64_t b = threadIdx.x; b < B; b += FIN) {
    float m = 0.0f;
#pragma unroll 8
    for (int c = 0; c < chunks; ++c) m += part[b * chunks + c];
    m *= inv_t;
    margin[b] = m;
    if (loss == nullptr) continue;
    const float z = beta * (m - (ref != nullptr ? ref[b] : 0.0f));
    const float tail = softplus_tail(z);
    // z as a factor last: 0 * infinity of an unsmoothed loss is not formed
    const float good = fmaxf(-z, 0.0f) + tail, bad = fmaxf(z, 0.0f) + tail;
    total += (z != z ? z : (1.0f - smoothing) * good + (smoothing > 0.0f ? smoothing * bad : 0.0f));
    const float e = __builtin_amdgcn_exp2f(-fabsf(z) * 1.44269504088896341f);
    // sigma(z) - 1 = -sigma(-z) is formed directly: the difference would cancel where z is large
    const float neg = z > 0.0f ? e / (1.0f + e) : 1.0f / (1.0f + e);
    coef[b] = (z != z ? z : smoothing - neg) * beta * inv_t / (float)B;
  }
  if (loss == nullptr) return;
  total = group_sum<FIN>(total, lds);
  if (threadIdx.x == 0) *loss = total / (float)B;
}

template <typename T>
__global__ __launch_bounds__(NT) void pref_grad_kernel(const T* __restrict__ q, const T* __restrict__ p,
                                                       const T* __restrict__ n, const float* __restrict__ coef,
                                                       const float* __restrict__ grad, int64_t V, int64_t chunks,
                                                       int64_t span, T* __restrict__ dq, T* __restrict__ dp,
                                                       T* __restrict__ dn) {
  constexpr int N = Vec<T>::N;
  const int64_t b = blockIdx.x / chunks, v0 = (int64_t)(blockIdx.x % chunks) * span, v1 = min(V, v0 + span);
  const int64_t base = b * V;
  const float c = coef[b] * *grad;
  if (V >= N) {
#pragma unroll 2
    for (int64_t v = v0 + threadIdx.x * N; v < v1; v += NT * N) {
      const int64_t at = base + min(v, V - N);
      const auto qv = load_any<T>(q + at), pv = load_any<T>(p + at), nv = load_any<T>(n + at);
      typename Vec<T>::type a, x, y;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        a[e] = from_f32<T>(c * (to_f32(pv[e]) - to_f32(nv[e])));
        const float w = c * to_f32(qv[e]);
        x[e] = from_f32<T>(w);
        y[e] = from_f32<T>(-w);
      }
      // A moved vector's lower elements are written twice, with the same values.
      store_any<T>(dq + at, a);
      store_any<T>(dp + at, x);
      store_any<T>(dn + at, y);
    }
  } else if ((int64_t)threadIdx.x < V) {
    const int64_t at = base + threadIdx.x;
    const float w = c * to_f32(q[at]);
    dq[at] = from_f32<T>(c * (to_f32(p[at]) - to_f32(n[at])));
    dp[at] = from_f32<T>(w);
    dn[at] = from_f32<T>(-w);
  }
}

int check(int64_t B, int64_t V, int dtype) {
  if (B < 1 || V < 1 || dtype < SPARTON_F32 || dtype > SPARTON_F16) return SPARTON_EINVAL;
  return B > kMaxGroups || V > INT32_MAX ? SPARTON_EUNSUPPORTED : SPARTON_OK;
}
bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int elem(int dtype) { return dtype == SPARTON_F32 ? 4 : 2; }

template <typename T>
void margins(const void* q, const void* p, const void* n, int64_t B, int64_t V, const Plan& pl, float* part, hipStream_t st) {
  hipLaunchKernelGGL(pref_margin_kernel<T>, dim3((unsigned)(B * pl.chunks)), dim3(NT), 0, st, (const T*)q, (const T*)p,
                     (const T*)n, V, pl.chunks, pl.span, part);
}
template <typename T>
void grads(const void* q, const void* p, const void* n, const float* coef, const float* grad, int64_t B, int64_t V,
           const Plan& pl, void* dq, void* dp, void* dn, hipStream_t st) {
  hipLaunchKernelGGL(pref_grad_kernel<T>, dim3((unsigned)(B * pl.chunks)), dim3(NT), 0, st, (const T*)q, (const T*)p,
                     (const T*)n, coef, grad, V, pl.chunks, pl.span, (T*)dq, (T*)dp, (T*)dn);
}

}  // namespace pref
}  // namespace sparton

using namespace sparton;

#define SPARTON_EXPORT extern "C" __attribute__((visibility("default")))

SPARTON_EXPORT size_t sparton_preference_workspace_bytes(int64_t B, int64_t V, int dtype) {
  if (pref::check(B, V, dtype) != SPARTON_OK) return 0;
  return (size_t)B * pref::margin_plan(B, V, pref::elem(dtype)).chunks * 4;
}

SPARTON_EXPORT int sparton_preference_fwd(const void* q, const void* pos, const void* neg, const float* ref_margin,
                                          int64_t B, int64_t V, float temperature, float beta, float smoothing,
                                          float* loss, float* margin, float* coef, void* workspace,
                                          size_t workspace_bytes, int dtype, void* stream) {
  const int rc = pref::check(B, V, dtype);
  if (rc == SPARTON_EINVAL) return rc;
  if (!(temperature > 0.0f) || isinf(temperature) || !(beta > 0.0f) || isinf(beta) || !(smoothing >= 0.0f) ||
      smoothing > 0.5f)
    return SPARTON_EINVAL;
  if (q == nullptr || pos == nullptr || neg == nullptr || margin == nullptr || (loss == nullptr) != (coef == nullptr))
    return SPARTON_EINVAL;
  if (rc != SPARTON_OK) return rc;
  const int es = pref::elem(dtype);
  if (!pref::aligned(q, es) || !pref::aligned(pos, es) || !pref::aligned(neg, es) || !pref::aligned(ref_margin, 4) ||
      !pref::aligned(loss, 4) || !pref::aligned(margin, 4) || !pref::aligned(coef, 4))
    return SPARTON_EALIGN;
  const pref::Plan pl = pref::margin_plan(B, V, es);
  if (workspace == nullptr || workspace_bytes < (size_t)B * pl.chunks * 4) return SPARTON_EWORKSPACE;
  if (!pref::aligned(workspace, 256)) return SPARTON_EALIGN;
  hipStream_t st = (hipStream_t)stream;
  float* part = (float*)workspace;
  if (dtype == SPARTON_BF16) pref::margins<bf16>(q, pos, neg, B, V, pl, part, st);
  else if (dtype == SPARTON_F16) pref::margins<f16>(q, pos, neg, B, V, pl, part, st);
  else pref::margins<float>(q, pos, neg, B, V, pl, part, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  hipLaunchKernelGGL(pref::pref_finish_kernel, dim3(1), dim3(pref::FIN), 0, st, (const float*)part, (int)pl.chunks,
                     ref_margin, B, 1.0f / temperature, beta, smoothing, loss, margin, coef);
  return (int)hipGetLastError();
}

SPARTON_EXPORT int sparton_preference_bwd(const void* q, const void* pos, const void* neg, const float* coef,
                                          const float* grad_loss, int64_t B, int64_t V, void* d_q, void* d_pos,
                                          void* d_neg, int dtype, void* stream) {
  const int rc = pref::check(B, V, dtype);
  if (rc == SPARTON_EINVAL) return rc;
  if (q == nullptr || pos == nullptr || neg == nullptr || coef == nullptr || grad_loss == nullptr || d_q == nullptr ||
      d_pos == nullptr || d_neg == nullptr)
    return SPARTON_EINVAL;
  if (rc != SPARTON_OK) return rc;
  const int es = pref::elem(dtype);
  if (!pref::aligned(q, es) || !pref::aligned(pos, es) || !pref::aligned(neg, es) || !pref::aligned(d_q, es) ||
      !pref::aligned(d_pos, es) || !pref::aligned(d_neg, es) || !pref::aligned(coef, 4) || !pref::aligned(grad_loss, 4))
    return SPARTON_EALIGN;
  const pref::Plan pl = pref::grad_plan(B, V, es);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SPARTON_BF16) pref::grads<bf16>(q, pos, neg, coef, grad_loss, B, V, pl, d_q, d_pos, d_neg, st);
  else if (dtype == SPARTON_F16) pref::grads<f16>(q, pos, neg, coef, grad_loss, B, V, pl, d_q, d_pos, d_neg, st);
  else pref::grads<float>(q, pos, neg, coef, grad_loss, B, V, pl, d_q, d_pos, d_neg, st);
  return (int)hipGetLastError();
}
