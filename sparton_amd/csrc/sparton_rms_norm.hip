// Root-mean-square norm of a backbone's rows, forward and backward, on gfx950, with the residual's addition:
//     h = x (+ r),  q = 1 / sqrt(mean(h^2) + eps) over the row,  y = h q gamma
//     8 bits:  s = max(max |y| / 448, 2^-126) over the row,  y8 = e4m3(y / s)
//     g = dy gamma,  dx = dr = q (g - h q mean(g h q)) + dh,  d gamma = sum over rows of dy h q
// The norm reads the unrounded sum h. What is stored of h (an output: the next layer's residual) is rounded to
// the rows' type, and the backward reads that, one row where x and r would be two: it enters dx through a mean
// over D, and adds to d gamma's error what rounding d gamma itself does. Both passes are bound by memory: a row
// is read once, held in registers between its sums and its output, and the next row's loads are in flight
// meanwhile.
//
// WPR waves work on one row (1 up to 1024 elements, then 4, then 8), each lane on NP vectors of 16 bytes, as in
// the LayerNorm (sparton_norm.hip). Every sum has a fixed order, so results are bitwise reproducible.
//
// Measured: 8192 x 4096 bf16 with a residual, forward 42 us (268 MB, 6.4 TB/s: more than a large copy's 5.1, as
// repeated runs probably find part of it cached), backward 45 and 4 for the columns' sums (201 MB, 4.1 TB/s), forward in e4m3
// 38. A few rows take 2.6, a launch. The backward of rows past 8192 spills 10 registers a lane in fp16 and 200 in
// fp32: 4096 x 16384 takes 86 us in bf16 (6.3 TB/s), 101 in fp16 and 508 in fp32 (2.1 TB/s).

#include <math.h>

#include <algorithm>

#include "sparton_common.h"
#include "sparton_rows.h"

namespace sparton {
namespace rms {

constexpr int kFwdWaves = 4;    // forward workgroups of 4 waves, or of the 8 waves of one row
constexpr int kBwdWaves = 8;
constexpr int kBwdBlocks = 256; // backward: one workgroup per CU, so that few partial sums are written
constexpr int64_t kMaxD = 16384;
constexpr float kE4m3Max = 448.0f;

struct Params {
  const void *x, *r, *dy, *dh, *gamma;
  const float* q;
  void *y, *h, *dx;
  float *q_out, *scale_out, *part;
  int64_t M;
  int D, vec_dtype;
  float eps, inv_d;
};

// VE values in e4m3, rounded to nearest even (none is above 448).
template <int VE> __device__ __forceinline__ void store_e4m3(uint8_t* p, const float* v) {
  if constexpr (VE == 1) {
    *p = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[0], 0, false);
  } else {
    typedef __attribute__((ext_vector_type(VE / 4))) int words;
    typedef words loose __attribute__((aligned(1)));
    words o;
#pragma unroll
    for (int i = 0; i < VE / 4; ++i) {
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
      o[i] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], lo, true);
    }
    *(loose*)p = o;
  }
}

// ---- forward ------------------------------------------------------------------------------
template <typename T, int VE, int NP, int WPR, bool BITS8>
__global__ __launch_bounds__(64 * (WPR > kFwdWaves ? WPR : kFwdWaves)) void rms_fwd_kernel(Params p) {
  constexpr int WAVES = WPR > kFwdWaves ? WPR : kFwdWaves, GROUPS = WAVES / WPR;
  __shared__ float slots[GROUPS][2][2][WPR];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int grp = wave / WPR, wir = wave % WPR, t = wir * 64 + lane;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  int64_t row = (int64_t)blockIdx.x * GROUPS + grp;
  // With several groups to a workgroup (WPR = 1) nothing is shared; otherwise every wave runs the
  // same rows, so barriers match.
  float ga[NP][VE];
  vec_t<T, VE> nx[NP], nr[NP];
  const auto fetch = [&](int64_t at) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const Place<VE> pl(VE * (t + 64 * WPR * i), p.D);
      nx[i] = load_any<T, VE>((const T*)p.x + at * p.D + pl.at);
      if (p.r != nullptr) nr[i] = load_any<T, VE>((const T*)p.r + at * p.D + pl.at);
    }
  };
  if (row < p.M) fetch(row);
#pragma unroll
  for (int i = 0; i < NP; ++i) vec_param<T, VE>(ga[i], p.gamma, p.vec_dtype, Place<VE>(VE * (t + 64 * WPR * i), p.D).at);
  for (int odd = 0; row < p.M; row += step, odd ^= 1) {
    float h[NP][VE];
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const Place<VE> pl(VE * (t + 64 * WPR * i), p.D);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        h[i][e] = to_f32(nx[i][e]);
        if (p.r != nullptr) h[i][e] += to_f32(nr[i][e]);
        s += e >= pl.own ? h[i][e] * h[i][e] : 0.0f;
      }
    }
    if (row + step < p.M) fetch(row + step);
    // consecutive rows alternate between two slots, so one barrier a sum will do
    const float q = rsqrtf(row_sum<WPR>(s, slots[grp][odd][0], wir) / (float)p.D + p.eps);
    float inv = 1.0f;
    if constexpr (BITS8) {
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) top = fmaxf(top, fabsf(h[i][e] * q * ga[i][e]));  // a moved vector's twice
      top = row_max<WPR>(top, slots[grp][odd][1], wir);
      const float scale = fmaxf(top / kE4m3Max, 0x1p-126f);
      inv = 1.0f / scale;
      if (t == 0) p.scale_out[row] = scale;
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const Place<VE> pl(VE * (t + 64 * WPR * i), p.D);
      const int64_t at = row * p.D + pl.at;
      float v[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) v[e] = h[i][e] * q * ga[i][e];
      if (pl.own == VE) continue;
      // A moved vector's lower elements are written twice, with the same value.
      if constexpr (BITS8) {
#pragma unroll
        for (int e = 0; e < VE; ++e) v[e] *= inv;
        store_e4m3<VE>((uint8_t*)p.y + at, v);
      } else {
        vec_t<T, VE> o;
#pragma unroll
        for (int e = 0; e < VE; ++e) o[e] = from_f32<T>(v[e]);
        store_any<T, VE>((T*)p.y + at, o);
      }
      if (p.h != nullptr) {
        vec_t<T, VE> o;
#pragma unroll
        for (int e = 0; e < VE; ++e) o[e] = from_f32<T>(h[i][e]);
        store_any<T, VE>((T*)p.h + at, o);
      }
    }
    if (t == 0 && p.q_out != nullptr) p.q_out[row] = q;
  }
}

// ---- backward -----------------------------------------------------------------------------
template <typename T, int VE, int NP, int WPR>
__global__ __launch_bounds__(64 * kBwdWaves) void rms_bwd_kernel(Params p) {
  constexpr int GROUPS = kBwdWaves / WPR, COLS = 64 * WPR * VE;  // columns of one of the NP steps
  __shared__ float slots[GROUPS][2][WPR];
  __shared__ __attribute__((aligned(16))) float cols[GROUPS][COLS];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int grp = wave / WPR, wir = wave % WPR, t = wir * 64 + lane;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  const int64_t row0 = (int64_t)blockIdx.x * GROUPS;
  // Rows in lockstep over the workgroup's groups (a group past the end repeats row M - 1 and keeps
  // nothing), so that barriers match.
  float ga[NP][VE], pg[NP][VE];
  vec_t<T, VE> nx[NP], ny[NP], nd[NP];
  float nq;
  const auto fetch = [&](int64_t row) {
    row = min(row, p.M - 1);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const Place<VE> pl(VE * (t + 64 * WPR * i), p.D);
      nx[i] = load_any<T, VE>((const T*)p.x + row * p.D + pl.at);
      ny[i] = load_any<T, VE>((const T*)p.dy + row * p.D + pl.at);
      if (p.dh != nullptr) nd[i] = load_any<T, VE>((const T*)p.dh + row * p.D + pl.at);
    }
    nq = p.q[row];
  };
  if (row0 < p.M) fetch(row0 + grp);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    vec_param<T, VE>(ga[i], p.gamma, p.vec_dtype, Place<VE>(VE * (t + 64 * WPR * i), p.D).at);
#pragma unroll
    for (int e = 0; e < VE; ++e) pg[i][e] = 0.0f;
  }
  int odd = 0;
  for (int64_t rb = row0; rb < p.M; rb += step, odd ^= 1) {
    const int64_t row = rb + grp;
    const bool in = row < p.M;
    float xh[NP][VE];
    vec_t<T, VE> cy[NP], cd[NP];
    float s = 0.0f;
    const float q = nq;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const Place<VE> pl(VE * (t + 64 * WPR * i), p.D);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float dy = to_f32(ny[i][e]);
        xh[i][e] = to_f32(nx[i][e]) * q;
        s += e >= pl.own ? dy * ga[i][e] * xh[i][e] : 0.0f;
        pg[i][e] += in ? dy * xh[i][e] : 0.0f;
      }
      cy[i] = ny[i];
      if (p.dh != nullptr) cd[i] = nd[i];
    }
    if (rb + step < p.M) fetch(rb + step + grp);
    const float c = row_sum<WPR>(s, slots[grp][odd], wir) * p.inv_d;
    if (in) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const Place<VE> pl(VE * (t + 64 * WPR * i), p.D);
        vec_t<T, VE> o;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          float d = q * (to_f32(cy[i][e]) * ga[i][e] - xh[i][e] * c);
          if (p.dh != nullptr) d += to_f32(cd[i][e]);
          o[e] = from_f32<T>(d);
        }
        if (pl.own < VE) store_any<T, VE>((T*)p.dx + row * p.D + pl.at, o);
      }
    }
  }
  // The groups' column sums added in group order, one step of columns at a time, into part[block][D].
  float* out = p.part + (int64_t)blockIdx.x * p.D;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VE; ++e) cols[grp][t * VE + e] = pg[i][e];
    __syncthreads();
    for (int j = threadIdx.x; j < COLS; j += 64 * kBwdWaves) {
      const int lane_at = j / VE * VE;
      const Place<VE> pl(i * COLS + lane_at, p.D);
      const int e = j - lane_at;
      if (e >= pl.own) {
        float a = 0.0f;
#pragma unroll
        for (int w = 0; w < GROUPS; ++w) a += cols[w][j];
        out[pl.at + e] = a;
      }
    }
  }
}

// ---- launches -----------------------------------------------------------------------------
enum Kind { kFwd, kFwd8, kBwd };

int waves_per_row(int64_t D) { return D <= 1024 ? 1 : D <= 2048 ? 4 : 8; }

int64_t bwd_blocks(int64_t M, int64_t D) {
  return std::min<int64_t>(kBwdBlocks, cdiv(M, kBwdWaves / waves_per_row(D)));
}

template <typename T, int VE, int NP, int WPR> void launch(const Params& p, Kind kind, hipStream_t st) {
  if (kind == kBwd) {
    hipLaunchKernelGGL((rms_bwd_kernel<T, VE, NP, WPR>), dim3((unsigned)bwd_blocks(p.M, p.D)), dim3(64 * kBwdWaves), 0,
                       st, p);
    return;
  }
  constexpr int WAVES = WPR > kFwdWaves ? WPR : kFwdWaves;
  // Past four workgroups of four waves a CU a wave takes several rows: it loads the weight once.
  const dim3 grid((unsigned)std::min<int64_t>(cdiv(p.M, WAVES / WPR), 1024 * kFwdWaves / WAVES));
  if (kind == kFwd8) hipLaunchKernelGGL((rms_fwd_kernel<T, VE, NP, WPR, true>), grid, dim3(64 * WAVES), 0, st, p);
  else hipLaunchKernelGGL((rms_fwd_kernel<T, VE, NP, WPR, false>), grid, dim3(64 * WAVES), 0, st, p);
}

template <typename T> void launch_t(const Params& p, Kind kind, hipStream_t st) {
  constexpr int VE = 16 / sizeof(T);
  constexpr int K = 8 / VE;  // fp32 rows take twice the vectors
  if (p.D < VE) return launch<T, 1, 1, 1>(p, kind, st);
  if (p.D <= 512) return launch<T, VE, K, 1>(p, kind, st);
  if (p.D <= 1024) return launch<T, VE, 2 * K, 1>(p, kind, st);
  if (p.D <= 2048) return launch<T, VE, K, 4>(p, kind, st);
  if (p.D <= 4096) return launch<T, VE, K, 8>(p, kind, st);
  if (p.D <= 8192) return launch<T, VE, 2 * K, 8>(p, kind, st);
  return launch<T, VE, 4 * K, 8>(p, kind, st);
}

void run(const Params& p, int dtype, Kind kind, hipStream_t st) {
  if (dtype == SPARTON_BF16) launch_t<bf16>(p, kind, st);
  else if (dtype == SPARTON_F16) launch_t<f16>(p, kind, st);
  else launch_t<float>(p, kind, st);
}

int check(int64_t M, int64_t D, int dtype, int vec_dtype) {
  if (M < 0 || D <= 0 || dtype < SPARTON_F32 || dtype > SPARTON_F16) return SPARTON_EINVAL;
  if (vec_dtype != SPARTON_F32 && vec_dtype != dtype) return SPARTON_EINVAL;
  return D > kMaxD || M > INT64_MAX / 4 / D ? SPARTON_EUNSUPPORTED : SPARTON_OK;
}

int forward(Kind kind, const void* x, const void* residual, const void* weight, int vec_dtype, float eps, void* y,
            float* scale, void* h, float* q, int64_t M, int64_t D, int dtype, hipStream_t st) {
  const int rc = check(M, D, dtype, vec_dtype);
  if (rc != SPARTON_OK) return rc;
  if (!(eps >= 0.0f) || isinf(eps)) return SPARTON_EINVAL;
  if (M == 0) return SPARTON_OK;
  if (x == nullptr || weight == nullptr || y == nullptr || (kind == kFwd8 && scale == nullptr)) return SPARTON_EINVAL;
  const uintptr_t es = dtype == SPARTON_F32 ? 4 : 2, vs = vec_dtype == SPARTON_F32 ? 4 : 2;
  if (!aligned(x, es) || !aligned(residual, es) || !aligned(y, kind == kFwd8 ? 1 : es) || !aligned(h, es) ||
      !aligned(weight, vs) || !aligned(q, 4) || !aligned(scale, 4))
    return SPARTON_EALIGN;
  Params p = {};
  p.x = x;
  p.r = residual;
  p.gamma = weight;
  p.vec_dtype = vec_dtype;
  p.eps = eps;
  p.y = y;
  p.h = h;
  p.q_out = q;
  p.scale_out = scale;
  p.M = M;
  p.D = (int)D;
  run(p, dtype, kind, st);
  return (int)hipGetLastError();
}

}  // namespace rms
}  // namespace sparton

using namespace sparton;

#define SPARTON_EXPORT extern "C" __attribute__((visibility("default")))

SPARTON_EXPORT int sparton_rms_norm_fwd(const void* x, const void* residual, const void* weight, int vec_dtype,
                                        float eps, void* y, void* h, float* rstd, int64_t M, int64_t D, int dtype,
                                        void* stream) {
  return rms::forward(rms::kFwd, x, residual, weight, vec_dtype, eps, y, nullptr, h, rstd, M, D, dtype,
                      (hipStream_t)stream);
}

SPARTON_EXPORT int sparton_rms_norm_fwd_quantized(const void* x, const void* residual, const void* weight, int vec_dtype,
                                             float eps, void* y, float* scale, void* h, int64_t M, int64_t D, int dtype,
                                             void* stream) {
  return rms::forward(rms::kFwd8, x, residual, weight, vec_dtype, eps, y, scale, h, nullptr, M, D, dtype,
                      (hipStream_t)stream);
}

SPARTON_EXPORT size_t sparton_rms_norm_workspace_bytes(int64_t M, int64_t D) {
  if (M <= 0 || D <= 0 || D > rms::kMaxD) return 0;
  return (size_t)rms::bwd_blocks(M, D) * D * 4;
}

SPARTON_EXPORT int sparton_rms_norm_bwd(const void* dy, const void* dh, const void* h, const void* weight, int vec_dtype,
                                        const float* rstd, void* dx, void* d_weight, void* workspace,
                                        size_t workspace_bytes, int64_t M, int64_t D, int dtype, void* stream) {
  const int rc = rms::check(M, D, dtype, vec_dtype);
  if (rc != SPARTON_OK) return rc;
  if (M > 0 && (dy == nullptr || h == nullptr || weight == nullptr || rstd == nullptr || dx == nullptr))
    return SPARTON_EINVAL;
  const uintptr_t es = dtype == SPARTON_F32 ? 4 : 2, vs = vec_dtype == SPARTON_F32 ? 4 : 2;
  if (!aligned(dy, es) || !aligned(dh, es) || !aligned(h, es) || !aligned(dx, es) || !aligned(weight, vs) ||
      !aligned(d_weight, vs) || !aligned(rstd, 4))
    return SPARTON_EALIGN;
  hipStream_t st = (hipStream_t)stream;
  int blocks = 0;
  if (M > 0) {
    if (workspace == nullptr || workspace_bytes < sparton_rms_norm_workspace_bytes(M, D)) return SPARTON_EWORKSPACE;
    if (!aligned(workspace, 256)) return SPARTON_EALIGN;
    rms::Params p = {};
    p.dy = dy;
    p.dh = dh;
    p.x = h;
    p.gamma = weight;
    p.vec_dtype = vec_dtype;
    p.q = rstd;
    p.dx = dx;
    p.part = (float*)workspace;
    p.M = M;
    p.D = (int)D;
    p.inv_d = 1.0f / (float)D;
    blocks = (int)rms::bwd_blocks(M, D);
    rms::run(p, dtype, rms::kBwd, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  if (d_weight == nullptr) return SPARTON_OK;
  hipLaunchKernelGGL(colsum_kernel, dim3((unsigned)cdiv(D, 64)), dim3(64 * kSumWaves), 0, st, (const float*)workspace,
                     blocks, (int)D, (int)D, d_weight, nullptr, vec_dtype);
  return (int)hipGetLastError();
}
