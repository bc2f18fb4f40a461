// LayerNorm of a backbone's rows, forward and backward, on gfx950, with the residual sum in front:
//     h = x (+ r),  mean and rstd = 1 / sqrt(var + eps) over the row,  xhat = (h - mean) rstd
//     y = xhat gamma (+ beta)
//     g = dy gamma,  dx = dr = rstd (g - mean(g) - xhat mean(g xhat))
//     d gamma = sum over rows of dy xhat,  d beta = sum over rows of dy
// h is summed in fp32 and recomputed by the backward from x and r: as many bytes as storing it would
// take, without its rounding. Both passes are bound by memory: a row is read once, held in registers
// between its sums and its output, and the next row's loads are in flight meanwhile.
//
// WPR waves work on one row (1 up to 1024 elements, then 4, then 8), each lane on NP vectors of 16
// bytes: lane t of the row's 64 WPR holds elements VE (t + 64 WPR p) .. + VE - 1. Rows need no
// alignment: global vector accesses take any address, and a row's last vector, where it would pass
// the end, is moved back to end with the row (its elements that a lower lane holds too count once).
// Every sum has a fixed order, so results are bitwise reproducible.
//
// Rows wider than a wave holds without spilling are shared by several waves, at the price of a barrier
// a sum; past 8192 elements the backward's eight spill all the same (14 registers a lane in bf16, 30 in
// fp16, 172 in fp32). bf16: 8192 x 768 with a residual, forward 10.0 us (3.8 TB/s), backward 12.6 (4.0) and
// 3.8 to add the column sums; 16385 x 4096, forward 55 to 62 us from box to box (4.4 to 4.8 TB/s), backward
// 76 to 80 (5.1 to 5.3) and 4.9. A copy reaches 4.9. 4096 x 16384 with a residual: backward 126 us in bf16
// (4.2 TB/s), 460 in fp32 (2.3).

#include <math.h>

#include <algorithm>

#include "sparton_common.h"
#include "sparton_rows.h"

namespace sparton {
namespace norm {

constexpr int kFwdWaves = 4;    // forward workgroups of 4 waves, or of the 8 waves of one row
constexpr int kBwdWaves = 8;
constexpr int kBwdBlocks = 256; // backward: one workgroup per CU, so that few partial sums are written
constexpr int64_t kMaxD = 16384;

struct Params {
  const void *x, *r, *dy, *gamma, *beta;
  const float *mean, *rstd;
  void *y, *dx;
  float *mean_out, *rstd_out, *part;
  int64_t M;
  int D, vec_dtype;
  float eps, inv_d;
};

// ---- forward ------------------------------------------------------------------------------
template <typename T, int VE, int NP, int WPR>
__global__ __launch_bounds__(64 * (WPR > kFwdWaves ? WPR : kFwdWaves)) void norm_fwd_kernel(Params p) {
  constexpr int WAVES = WPR > kFwdWaves ? WPR : kFwdWaves, GROUPS = WAVES / WPR;
  __shared__ float slots[GROUPS][2][WPR];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int grp = wave / WPR, wir = wave % WPR, t = wir * 64 + lane;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  int64_t row = (int64_t)blockIdx.x * GROUPS + grp;
  // With several groups to a workgroup (WPR = 1) nothing is shared; otherwise every wave runs the
  // same rows, so barriers match.
  float ga[NP][VE], be[NP][VE];
  vec_t<T, VE> nx[NP], nr[NP];
#pragma unroll
  for (int q = 0; q < NP; ++q) {
    const Place<VE> pl(VE * (t + 64 * WPR * q), p.D);
    if (row < p.M) {
      nx[q] = load_any<T, VE>((const T*)p.x + row * p.D + pl.at);
      if (p.r != nullptr) nr[q] = load_any<T, VE>((const T*)p.r + row * p.D + pl.at);
    }
    vec_param<T, VE>(ga[q], p.gamma, p.vec_dtype, pl.at);
    if (p.beta != nullptr) vec_param<T, VE>(be[q], p.beta, p.vec_dtype, pl.at);
    else
#pragma unroll
      for (int e = 0; e < VE; ++e) be[q][e] = 0.0f;
  }
  for (; row < p.M; row += step) {
    float h[NP][VE];
    float s = 0.0f;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const Place<VE> pl(VE * (t + 64 * WPR * q), p.D);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        h[q][e] = to_f32(nx[q][e]);
        if (p.r != nullptr) h[q][e] += to_f32(nr[q][e]);
        s += e >= pl.own ? h[q][e] : 0.0f;
      }
    }
    if (row + step < p.M) {
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        const Place<VE> pl(VE * (t + 64 * WPR * q), p.D);
        nx[q] = load_any<T, VE>((const T*)p.x + (row + step) * p.D + pl.at);
        if (p.r != nullptr) nr[q] = load_any<T, VE>((const T*)p.r + (row + step) * p.D + pl.at);
      }
    }
    // divided, not multiplied by 1/D: a constant row's mean is then that constant, where its sum is exact
    const float mu = row_sum<WPR>(s, slots[grp][0], wir) / (float)p.D;
    float v = 0.0f;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const Place<VE> pl(VE * (t + 64 * WPR * q), p.D);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        h[q][e] -= mu;
        v += e >= pl.own ? h[q][e] * h[q][e] : 0.0f;
      }
    }
    const float rs = rsqrtf(row_sum<WPR>(v, slots[grp][1], wir) / (float)p.D + p.eps);
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const Place<VE> pl(VE * (t + 64 * WPR * q), p.D);
      vec_t<T, VE> o;
#pragma unroll
      for (int e = 0; e < VE; ++e) o[e] = from_f32<T>(fmaf(h[q][e] * rs, ga[q][e], be[q][e]));
      // A moved vector's lower elements are written twice, with the same value.
      if (pl.own < VE) store_any<T, VE>((T*)p.y + row * p.D + pl.at, o);
    }
    if (t == 0 && p.mean_out != nullptr) {
      p.mean_out[row] = mu;
      p.rstd_out[row] = rs;
    }
  }
}

// ---- backward -----------------------------------------------------------------------------
template <typename T, int VE, int NP, int WPR>
__global__ __launch_bounds__(64 * kBwdWaves) void norm_bwd_kernel(Params p) {
  constexpr int GROUPS = kBwdWaves / WPR, COLS = 64 * WPR * VE;  // columns of one of the NP steps
  __shared__ float slots[GROUPS][2][2][WPR];
  __shared__ __attribute__((aligned(16))) float cols[GROUPS][COLS];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int grp = wave / WPR, wir = wave % WPR, t = wir * 64 + lane;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  const int64_t row0 = (int64_t)blockIdx.x * GROUPS;
  // Rows in lockstep over the workgroup's groups (a group past the end repeats row M - 1 and keeps
  // nothing), so that barriers match.
  float ga[NP][VE], pg[NP][VE], pb[NP][VE];
  vec_t<T, VE> nx[NP], nr[NP], ny[NP];
  float nmu, nrs;
  const auto fetch = [&](int64_t row) {
    row = min(row, p.M - 1);
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const Place<VE> pl(VE * (t + 64 * WPR * q), p.D);
      nx[q] = load_any<T, VE>((const T*)p.x + row * p.D + pl.at);
      ny[q] = load_any<T, VE>((const T*)p.dy + row * p.D + pl.at);
      if (p.r != nullptr) nr[q] = load_any<T, VE>((const T*)p.r + row * p.D + pl.at);
    }
    nmu = p.mean[row];
    nrs = p.rstd[row];
  };
  if (row0 < p.M) fetch(row0 + grp);
#pragma unroll
  for (int q = 0; q < NP; ++q) {
    const Place<VE> pl(VE * (t + 64 * WPR * q), p.D);
    vec_param<T, VE>(ga[q], p.gamma, p.vec_dtype, pl.at);
#pragma unroll
    for (int e = 0; e < VE; ++e) pg[q][e] = pb[q][e] = 0.0f;
  }
  int odd = 0;
  for (int64_t rb = row0; rb < p.M; rb += step, odd ^= 1) {
    const int64_t row = rb + grp;
    const bool in = row < p.M;
    float xh[NP][VE];
    vec_t<T, VE> cy[NP];
    float s1 = 0.0f, s2 = 0.0f;
    const float mu = nmu, rs = nrs;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const Place<VE> pl(VE * (t + 64 * WPR * q), p.D);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        float h = to_f32(nx[q][e]);
        if (p.r != nullptr) h += to_f32(nr[q][e]);
        const float dy = to_f32(ny[q][e]), g = dy * ga[q][e];
        xh[q][e] = (h - mu) * rs;
        s1 += e >= pl.own ? g : 0.0f;
        s2 += e >= pl.own ? g * xh[q][e] : 0.0f;
        pg[q][e] += in ? dy * xh[q][e] : 0.0f;
        pb[q][e] += in ? dy : 0.0f;
      }
      cy[q] = ny[q];
    }
    if (rb + step < p.M) fetch(rb + step + grp);
    float c1, c2;
    if constexpr (WPR == 1) {
      c1 = wave_sum(s1) * p.inv_d;
      c2 = wave_sum(s2) * p.inv_d;
    } else {
      s1 = wave_sum(s1);
      s2 = wave_sum(s2);
      float(*slot)[WPR] = slots[grp][odd];
      if (lane == 0) {
        slot[0][wir] = s1;
        slot[1][wir] = s2;
      }
      __syncthreads();
      c1 = c2 = 0.0f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) {
        c1 += slot[0][w];
        c2 += slot[1][w];
      }
      c1 *= p.inv_d;
      c2 *= p.inv_d;
    }
    if (in) {
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        const Place<VE> pl(VE * (t + 64 * WPR * q), p.D);
        vec_t<T, VE> o;
#pragma unroll
        for (int e = 0; e < VE; ++e) o[e] = from_f32<T>(rs * (to_f32(cy[q][e]) * ga[q][e] - c1 - xh[q][e] * c2));
        if (pl.own < VE) store_any<T, VE>((T*)p.dx + row * p.D + pl.at, o);
      }
    }
  }
  // The groups' column sums added in group order, one step of columns at a time, into part[block][2][D].
  float* out = p.part + (int64_t)blockIdx.x * 2 * p.D;
#pragma unroll
  for (int q = 0; q < NP; ++q)
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < VE; ++e) cols[grp][t * VE + e] = which == 0 ? pg[q][e] : pb[q][e];
      __syncthreads();
      for (int i = threadIdx.x; i < COLS; i += 64 * kBwdWaves) {
        const int lane_at = i / VE * VE;
        const Place<VE> pl(q * COLS + lane_at, p.D);
        const int e = i - lane_at;
        if (e >= pl.own) {
          float a = 0.0f;
#pragma unroll
          for (int w = 0; w < GROUPS; ++w) a += cols[w][i];
          out[which * p.D + pl.at + e] = a;
        }
      }
    }
}

// ---- launches -----------------------------------------------------------------------------
int waves_per_row(int64_t D) { return D <= 1024 ? 1 : D <= 2048 ? 4 : 8; }

int64_t bwd_blocks(int64_t M, int64_t D) {
  return std::min<int64_t>(kBwdBlocks, cdiv(M, kBwdWaves / waves_per_row(D)));
}

template <typename T, int VE, int NP, int WPR> void launch(const Params& p, bool bwd, hipStream_t st) {
  if (bwd) {
    hipLaunchKernelGGL((norm_bwd_kernel<T, VE, NP, WPR>), dim3((unsigned)bwd_blocks(p.M, p.D)), dim3(64 * kBwdWaves), 0,
                       st, p);
    return;
  }
  constexpr int WAVES = WPR > kFwdWaves ? WPR : kFwdWaves;
  // Past four workgroups of four waves a CU a wave takes several rows: it loads weight and bias once
  // (8192 x 768 in bf16: 10.0 us, with eight workgroups a CU and parameters read one by one 20.6).
  const int64_t groups = std::min<int64_t>(cdiv(p.M, WAVES / WPR), 1024 * kFwdWaves / WAVES);
  hipLaunchKernelGGL((norm_fwd_kernel<T, VE, NP, WPR>), dim3((unsigned)groups), dim3(64 * WAVES), 0, st, p);
}

template <typename T> void launch_t(const Params& p, bool bwd, hipStream_t st) {
  constexpr int VE = 16 / sizeof(T);
  constexpr int K = 8 / VE;  // fp32 rows take twice the vectors
  if (p.D < VE) return launch<T, 1, 1, 1>(p, bwd, st);
  if (p.D <= 512) return launch<T, VE, K, 1>(p, bwd, st);
  if (p.D <= 1024) return launch<T, VE, 2 * K, 1>(p, bwd, st);
  if (p.D <= 2048) return launch<T, VE, K, 4>(p, bwd, st);
  if (p.D <= 4096) return launch<T, VE, K, 8>(p, bwd, st);
  if (p.D <= 8192) return launch<T, VE, 2 * K, 8>(p, bwd, st);
  return launch<T, VE, 4 * K, 8>(p, bwd, st);
}

void run(const Params& p, int dtype, bool bwd, hipStream_t st) {
  if (dtype == SPARTON_BF16) launch_t<bf16>(p, bwd, st);
  else if (dtype == SPARTON_F16) launch_t<f16>(p, bwd, st);
  else launch_t<float>(p, bwd, st);
}

int check(int64_t M, int64_t D, int dtype, int vec_dtype) {
  if (M < 0 || D <= 0 || dtype < SPARTON_F32 || dtype > SPARTON_F16) return SPARTON_EINVAL;
  if (vec_dtype != SPARTON_F32 && vec_dtype != dtype) return SPARTON_EINVAL;
  return D > kMaxD || M > INT64_MAX / 4 / D ? SPARTON_EUNSUPPORTED : SPARTON_OK;
}

}  // namespace norm
}  // namespace sparton

using namespace sparton;

#define SPARTON_EXPORT extern "C" __attribute__((visibility("default")))

SPARTON_EXPORT int sparton_layer_norm_fwd(const void* x, const void* residual, const void* weight, const void* bias,
                                          int vec_dtype, float eps, void* y, float* mean, float* rstd, int64_t M,
                                          int64_t D, int dtype, void* stream) {
  const int rc = norm::check(M, D, dtype, vec_dtype);
  if (rc != SPARTON_OK) return rc;
  if (!(eps >= 0.0f) || isinf(eps)) return SPARTON_EINVAL;
  if (M == 0) return SPARTON_OK;
  if (x == nullptr || weight == nullptr || y == nullptr || (mean == nullptr) != (rstd == nullptr)) return SPARTON_EINVAL;
  const uintptr_t es = dtype == SPARTON_F32 ? 4 : 2, vs = vec_dtype == SPARTON_F32 ? 4 : 2;
  if (!aligned(x, es) || !aligned(residual, es) || !aligned(y, es) || !aligned(weight, vs) ||
      !aligned(bias, vs) || !aligned(mean, 4) || !aligned(rstd, 4))
    return SPARTON_EALIGN;
  norm::Params p = {};
  p.x = x;
  p.r = residual;
  p.gamma = weight;
  p.beta = bias;
  p.vec_dtype = vec_dtype;
  p.eps = eps;
  p.y = y;
  p.mean_out = mean;
  p.rstd_out = rstd;
  p.M = M;
  p.D = (int)D;
  p.inv_d = 1.0f / (float)D;
  norm::run(p, dtype, false, (hipStream_t)stream);
  return (int)hipGetLastError();
}

SPARTON_EXPORT size_t sparton_layer_norm_workspace_bytes(int64_t M, int64_t D) {
  if (M <= 0 || D <= 0 || D > norm::kMaxD) return 0;
  return (size_t)norm::bwd_blocks(M, D) * 2 * D * 4;
}

SPARTON_EXPORT int sparton_layer_norm_bwd(const void* dy, const void* x, const void* residual, const void* weight,
                                          int vec_dtype, const float* mean, const float* rstd, void* dx,
                                          void* d_weight, void* d_bias, void* workspace, size_t workspace_bytes,
                                          int64_t M, int64_t D, int dtype, void* stream) {
  const int rc = norm::check(M, D, dtype, vec_dtype);
  if (rc != SPARTON_OK) return rc;
  if (M > 0 && (dy == nullptr || x == nullptr || weight == nullptr || mean == nullptr || rstd == nullptr || dx == nullptr))
    return SPARTON_EINVAL;
  const uintptr_t es = dtype == SPARTON_F32 ? 4 : 2, vs = vec_dtype == SPARTON_F32 ? 4 : 2;
  if (!aligned(dy, es) || !aligned(x, es) || !aligned(residual, es) || !aligned(dx, es) ||
      !aligned(weight, vs) || !aligned(d_weight, vs) || !aligned(d_bias, vs) ||
      !aligned(mean, 4) || !aligned(rstd, 4))
    return SPARTON_EALIGN;
  hipStream_t st = (hipStream_t)stream;
  int blocks = 0;
  if (M > 0) {
    const size_t need = sparton_layer_norm_workspace_bytes(M, D);
    if (workspace == nullptr || workspace_bytes < need) return SPARTON_EWORKSPACE;
    if (!aligned(workspace, 256)) return SPARTON_EALIGN;
    norm::Params p = {};
    p.dy = dy;
    p.x = x;
    p.r = residual;
    p.gamma = weight;
    p.vec_dtype = vec_dtype;
    p.mean = mean;
    p.rstd = rstd;
    p.dx = dx;
    p.part = (float*)workspace;
    p.M = M;
    p.D = (int)D;
    p.inv_d = 1.0f / (float)D;
    blocks = (int)norm::bwd_blocks(M, D);
    norm::run(p, dtype, true, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  if (d_weight == nullptr && d_bias == nullptr) return SPARTON_OK;
  hipLaunchKernelGGL(colsum_kernel, dim3((unsigned)cdiv(2 * D, 64)), dim3(64 * kSumWaves), 0, st,
                     (const float*)workspace, blocks, (int)D, 2 * (int)D, d_weight, d_bias, vec_dtype);
  return (int)hipGetLastError();
}
