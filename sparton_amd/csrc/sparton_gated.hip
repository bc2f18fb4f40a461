// Gated feed-forward product, forward and backward, on gfx950:
//     g = x Wg' + bg,  u = x Wu' + bu,  h = act(g) u             x [M, D], Wg and Wu [F, D], h [M, F]
//     du = dh act(g),  dg = dh u act'(g)
//     dx = dg Wg + du Wu,  dWg = dg' x,  dWu = du' x,  db = column sums of dg and du
// and the forward on e4m3 rows and weights with a scale a row.
//
// One kernel runs every product. A workgroup's tile is BQ rows by BP columns of the result, its inner dimension
// streams through LDS in slabs of 128 bytes (rows in two stages, columns in three), copied there directly from memory. A wave holds its part as
// 32x32 MFMA results in transposed form: a lane is a row of the result, and its registers hold groups of four
// consecutive columns, which it stores as one vector. The forward's columns are 32 of the gate, 32 of the up
// projection and so on, so g and u of one element meet in one lane.
//
// An operand whose memory runs along the inner dimension (x and the weights forward, dg and du for dx) is staged as
// rows of 128 bytes; one that runs across it (the weights for dx, everything for dW) as it lies, 64 rows of BQ or BP
// columns, and read with the transposing LDS loads (fp32: element by element). Nothing is transposed in memory.
// Both have their 16-byte chunks XORed so that the reads spread over all banks. What lies past an operand's end is
// given an address past the buffer's, which reads as zero.
//
// The 8-bit matrix instructions add the products of eight neighbours with about 14 bits below the largest one's power
// of two (what is further below is dropped), and such sums in fp32. The rows' own rounding to e4m3, 2^-4, is far above that.
//
// Between forward and backward g and u are kept in fp32: in 16 bits their rounding, on top of that of dg and du to
// the matrix instructions' operands, would add to the gradients' error. In fp16, dg and du have fp16's range, as dh has.
//
// Measured, 8192 x 4096 x 11264 bf16 (M, D, F): forward 1217 us with g and u stored (1242 TFLOP/s), dg and du 254 to 275
// (5.1 TB/s), dx 1104 (1370), dW 1183 with its join (1278): a library's large products reach 1386 to 1581. The matrix
// unit is busy for 71, 83 and 75% of the CUs' cycles, at about 1.7 GHz. The forward in e4m3 589 to 690. What is lost is
// at a tile's ends: about 10 us of each round of tiles beside 1.5 a slab. 8192 x 768 x 2048 bf16, gelu: 73, 34, 55 and
// 66. 1000 x 768 x 2051 fp32: forward 97 to 104, dx 65, dW 75.

#include <math.h>

#include <algorithm>
#include <type_traits>

#include "sparton_common.h"
#include "sparton_rows.h"

namespace sparton {
namespace gated {

constexpr int kSlab = 128;  // bytes of the inner dimension
constexpr int kGroupQ = 8;  // row tiles that share the weights' tiles while both are in an XCD's L2
constexpr uint64_t kMaxThreads = 1ull << 32;  // a launch holds fewer (past that, workgroups were left out)

struct e4m3 {
  uint8_t bits;
};

typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) int i32x8;

// ---- activations --------------------------------------------------------------------------
// On the hardware's base-2 exponential and reciprocal (1 ulp each); the exponents' own rounding makes exp(-x) off by
// x 2^-24.
__device__ __forceinline__ float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * -1.44269504088896341f); }
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_neg(x)); }

// The normal distribution's integral up to g: with x = |g| / sqrt(2) and t = 1 / (1 + 0.4 x),
//     erfc(x) / 2 = exp(-x^2) t Q(t),   Q(t) = erfc(x) exp(x^2) / (2 t), a smooth function on (0, 1],
// here its polynomial of degree 10, fitted for the least relative error (4.2e-8, with the coefficients and the factor
// 0.4 / sqrt(2) in fp32, up to |g| = 13; the coefficients' share is 2.0e-8), below fp32's half step. e: exp(-g^2 / 2).
__device__ __forceinline__ float normal_below(float g, float e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.28284271247461901f, fabsf(g), 1.0f));
  float q = -0.014607510529458523f;
  q = fmaf(q, t, 0.07022310048341751f);
  q = fmaf(q, t, -0.11776304990053177f);
  q = fmaf(q, t, 0.06877996772527695f);
  q = fmaf(q, t, -0.023447012528777122f);
  q = fmaf(q, t, 0.04195791855454445f);
  q = fmaf(q, t, 0.05950424075126648f);
  q = fmaf(q, t, 0.08586962521076202f);
  q = fmaf(q, t, 0.10380686819553375f);
  q = fmaf(q, t, 0.11283793300390244f);
  q = fmaf(q, t, 0.11283791810274124f);
  const float w = t * q * e;
  return g < 0.0f ? w : 1.0f - w;
}

// act(g), and its derivative where it is asked for.
template <int ACT, bool GRAD> __device__ __forceinline__ float activate(float g, float* d) {
  if constexpr (ACT == SPARTON_SILU) {
    const float s = sigmoid(g);
    if (GRAD) *d = s * fmaf(g, 1.0f - s, 1.0f);
    return g * s;
  } else if constexpr (ACT == SPARTON_GELU) {
    const float e = exp_neg(0.5f * g * g), c = normal_below(g, e);
    if (GRAD) *d = fmaf(g * e, 0.39894228040143268f, c);
    return g * c;
  } else if constexpr (ACT == SPARTON_GELU_TANH) {  // (1 + tanh(z)) / 2 = sigmoid(2 z)
    const float s = sigmoid(g * fmaf(0.071354816272600243f, g * g, 1.5957691216057308f));
    if (GRAD) *d = fmaf(g * s * (1.0f - s), fmaf(0.21406444881780073f, g * g, 1.5957691216057308f), s);
    return g * s;
  } else {
    if (GRAD) *d = g > 0.0f ? 1.0f : 0.0f;
    return g > 0.0f || g != g ? g : 0.0f;
  }
}
// f(std::integral_constant<int, act>)
template <typename F> __device__ __forceinline__ void with_activation(int act, const F& f) {
  switch (act) {  // uniform
    case SPARTON_SILU: return f(std::integral_constant<int, SPARTON_SILU>());
    case SPARTON_GELU: return f(std::integral_constant<int, SPARTON_GELU>());
    case SPARTON_GELU_TANH: return f(std::integral_constant<int, SPARTON_GELU_TANH>());
    default: return f(std::integral_constant<int, SPARTON_RELU>());
  }
}

// ---- matrix instructions ------------------------------------------------------------------
// A step's operand: CH chunks of 16 bytes a lane. Lane l holds row (or column) l % 32, and of each 32 bytes of the
// inner dimension the half l / 32.
template <typename T> constexpr int kCh = 1;
template <> constexpr int kCh<e4m3> = 2;
template <typename T> struct Frag {
  u32x4 c[kCh<T>];
};

__device__ __forceinline__ void mma(f32x16& d, const Frag<bf16>& a, const Frag<bf16>& b) {
  d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a.c[0]), __builtin_bit_cast(bf16x8, b.c[0]), d, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16& d, const Frag<f16>& a, const Frag<f16>& b) {
  d = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a.c[0]), __builtin_bit_cast(f16x8, b.c[0]), d, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16& d, const Frag<float>& a, const Frag<float>& b) {
  const f32x4 x = __builtin_bit_cast(f32x4, a.c[0]), y = __builtin_bit_cast(f32x4, b.c[0]);
#pragma unroll
  for (int e = 0; e < 4; ++e) d = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], d, 0, 0, 0);
}
__device__ __forceinline__ i32x8 wide(const Frag<e4m3>& f) {
  return __builtin_shufflevector(__builtin_bit_cast(i32x4, f.c[0]), __builtin_bit_cast(i32x4, f.c[1]), 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ void mma(f32x16& d, const Frag<e4m3>& a, const Frag<e4m3>& b) {
  d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(a), wide(b), d, 0, 0, 0, 0, 0, 0);
}

// ---- operands -----------------------------------------------------------------------------
// One operand of a product: n rows (columns, where it lies across the inner dimension) that start `ld` bytes apart.
// b1: the second half of the inner dimension (dx), or the rows that take turns with b0's (forward).
struct Side {
  const char *b0, *b1;
  int64_t ld, n;
};

__device__ __forceinline__ int swizzle_rows(int row) { return (row & 7) ^ ((row >> 3) & 1); }

// A wave's share of copying one operand's slabs: R rows of 128 bytes, or 128 / sizeof(T) rows of R elements (KM), by
// NW waves, 64 chunks of 16 bytes a copy. PAIR: rows 64 k .. + 31 of b0, rows 64 k + 32 .. + 63 of b1.
template <typename T, bool KM, int R, int NW, bool PAIR> struct Copy {
  static constexpr int E = sizeof(T), N = R / 8 / NW, CPR = KM ? R * E / 16 : 8;
  static_assert(R % (8 * NW) == 0, "every wave copies as much");
  static_assert(!PAIR || NW == 4, "the waves' copies i are rows 32 i .. + 31");
  static constexpr uint32_t kNowhere = 0xc0000000u;
  uint32_t off[N];
  int at;  // KC: byte of the slab; KM: its row
  const char *b0, *b1;
  int64_t step;
  __device__ __forceinline__ void init(const Side& s, int64_t first) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if constexpr (!KM) {
      at = ((lane & 7) ^ (lane >> 3) ^ (w & 1)) * 16;
      step = kSlab;
      b0 = s.b0 + first * s.ld;
      b1 = s.b1 + first * s.ld;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = 8 * (w + NW * i) + (lane >> 3), row = PAIR ? (r >> 6) * 32 + (r & 31) : r;
        off[i] = first + row < s.n ? (uint32_t)(row * s.ld + at) : kNowhere;
      }
    } else {
      const int c = w * 64 + lane;
      at = c / CPR;
      step = (int64_t)(kSlab / E) * s.ld;
      b0 = s.b0 + first * E;
      b1 = s.b1 + first * E;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int row = at + i * (NW * 64 / CPR);
        const int chunk = c % CPR ^ (E == 2 ? (row & 3) << 2 : ((row >> 2) & 1) << 3);
        off[i] = first + chunk * (16 / E) < s.n ? (uint32_t)(row * s.ld + chunk * 16) : kNowhere;
      }
    }
  }
  // What the copies of one slab share.
  struct Slab {
    const char *p0, *p1;
    int64_t left;
  };
  // Slab k of one half, of whose inner dimension `left` elements (none or fewer: zeros) are left.
  __device__ __forceinline__ Slab slab(int half, int k, int64_t left) const {
    const char* p0 = (!PAIR && half ? b1 : b0) + k * step;
    return Slab{p0, PAIR ? b1 + k * step : p0, left};
  }
  // Copy i of this wave, into LDS from `to` (the wave's first chunk) on.
  __device__ __forceinline__ void issue(const Slab& s, int i, uint32_t to) const {
    const bool in = KM ? at + i * (NW * 64 / CPR) < s.left : at < s.left * E;
    const uint32_t o = in ? off[i] : kNowhere, dst = to + (uint32_t)(i * NW) * 1024u;
    const uintptr_t from = (uintptr_t)(PAIR && (i & 1) ? s.p1 : s.p0);  // 32 rows a copy of all four waves
    u32x4 r;  // the compiler does not see that these are the same in every lane
    r[0] = __builtin_amdgcn_readfirstlane((uint32_t)from);
    r[1] = __builtin_amdgcn_readfirstlane((uint32_t)(from >> 32));
    r[2] = 0x80000000u;
    r[3] = 0x00020000u;
    // The compiler would wait for a copy it knows of before any LDS read; these are waited for at the slab's end. It
    // allocates m0 to nothing and warns of it as a reserved register; named here, what it may write there itself right
    // before an instruction of its own keeps clear of this.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(dst), "v"(o), "s"(r) : "m0");
#pragma clang diagnostic pop
  }
};

// Where a lane's fragments lie in a slab: J blocks of 32 rows (columns) from block `blk` on.
template <typename T, bool KM, int R, int J> struct Read {
  static constexpr int E = sizeof(T);
  const char* p[KM ? J : 4];
  __device__ __forceinline__ void init(int blk) {
    const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
    if constexpr (!KM) {
#pragma unroll
      for (int s = 0; s < 4; ++s)
        p[s] = (const char*)(uintptr_t)((blk * 32 + l32) * kSlab + ((2 * s + h) ^ swizzle_rows(l32)) * 16);
    } else if constexpr (E == 2) {
      const int q = lane & 15, kk = q >> 2;
#pragma unroll
      for (int j = 0; j < J; ++j)
        p[j] = (const char*)(uintptr_t)((8 * h + kk) * (R * 2) + (((blk + j) * 4) ^ (kk << 2)) * 16 + ((lane >> 4) & 1) * 32 +
                                        (q & 3) * 8);
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j)
        p[j] = (const char*)(uintptr_t)(4 * h * (R * 4) + (((blk + j) * 8) ^ (h << 3)) * 16 + l32 * 4);
    }
  }
  // Block j's operand of step s, of the slab at `slab`.
  __device__ __forceinline__ Frag<T> get(const char* slab, int j, int s) const {
    Frag<T> f;
    if constexpr (!KM) {
#pragma unroll
      for (int c = 0; c < kCh<T>; ++c) f.c[c] = *(const u32x4*)(slab + (uintptr_t)p[s * kCh<T> + c] + j * 32 * kSlab);
    } else if constexpr (E == 2) {
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const char* at = slab + (uintptr_t)p[j] + s * 16 * (R * 2);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 4 * (R * 2)));
      f.c[0] = __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const char* at = slab + (uintptr_t)p[j] + s * 8 * (R * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) f.c[0][e] = *(const uint32_t*)(at + e * (R * 4));
    }
    return f;
  }
};

// ---- the product --------------------------------------------------------------------------
struct Params {
  Side q, p;              // rows and columns of the result
  int64_t K;              // inner dimension of a half, in elements
  int half_slabs, slabs;  // of one half, and of all halves
  int tq, tp;             // tiles of rows and columns
  int whole;              // tiles that one workgroup makes; of the others, `splits` share the inner dimension
  int splits, per_split;
  // plain results: rows [0, q.n) of out; `turns` problems beside each other. part: [tile - whole][split][BQ][BP]
  void* out[2];
  const char* q_turn;
  float* part;
  int turns;
  // the gated result
  void* h;
  float *g, *u;
  const void *bg, *bu;
  const float *sx, *sg, *su;
  int act;
};

// A workgroup's tile. Tiles walk kGroupQ row tiles before the next column tile. Consecutive workgroups go to the eight
// XCDs in turn: each XCD takes a run of the whole tiles, so that what it has in flight shares operands in its L2. The
// workgroups that share tiles come last.
struct Place {
  int q, p, split, turn, shared;  // shared: the tile's place among those that are, or -1
};
__device__ __forceinline__ Place tile_of(const Params& a, int i) {
  Place r = {};
  r.turn = i / (a.tq * a.tp);
  i -= r.turn * a.tq * a.tp;
  const int group = i / (kGroupQ * a.tp), first = group * kGroupQ, rows = min(kGroupQ, a.tq - first);
  i -= first * a.tp;
  r.p = i / rows;
  r.q = first + i - r.p * rows;
  return r;
}
// Workgroup w's place in n, an XCD's ones in a run.
__device__ __forceinline__ int in_runs(int w, int n) {
  const int x = w & 7, per = n >> 3, more = n & 7;
  return x * per + min(x, more) + (w >> 3);
}
__device__ __forceinline__ Place place_of(const Params& a) {
  const int w = blockIdx.x;
  if (w < a.whole) {
    Place r = tile_of(a, in_runs(w, a.whole));
    r.shared = -1;
    return r;
  }
  const int rest = a.tq * a.tp * a.turns - a.whole, j = in_runs(w - a.whole, rest * a.splits);  // `whole`: rounds of CUs
  Place r = tile_of(a, a.whole + j % rest);
  r.shared = j % rest;
  r.split = j / rest;
  return r;
}

// N consecutive columns of a result's row, of which `n` are there.
template <typename T, int N> __device__ __forceinline__ void store_n(T* p, const float* v, int64_t n) {
  constexpr int V = N * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : N;
#pragma unroll
  for (int k = 0; k < N; k += V) {
    if (n >= k + V) {
      vec_t<T, V> o;
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = from_f32<T>(v[k + e]);
      store_any<T, V>(p + k, o);
    } else {
#pragma unroll
      for (int e = 0; e < V - 1; ++e)
        if (k + e < n) p[k + e] = from_f32<T>(v[k + e]);
    }
  }
}

// A lane's four columns of the gated result: what is the same in every row, read once.
template <typename T, typename O> struct Columns {
  int64_t col, left;  // columns from col on that are there: none for 0 or fewer
  float bg[4], bu[4], sg[4], su[4];
  __device__ __forceinline__ void init(const Params& a, int64_t col_) {
    col = col_;
    left = a.p.n - col;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t f = min(col + e, a.p.n - 1);
      bg[e] = a.bg != nullptr ? to_f32(((const O*)a.bg)[f]) : 0.0f;
      bu[e] = a.bu != nullptr ? to_f32(((const O*)a.bu)[f]) : 0.0f;
      if constexpr (sizeof(T) == 1) {
        sg[e] = a.sg[f];
        su[e] = a.su[f];
      }
    }
  }
  // One row of them from the products' sums (8 bits: before the scales): h, and g and u where they are kept, at `at`
  // elements from the pointers. WHOLE: all four columns are there.
  template <int ACT, bool WHOLE>
  __device__ __forceinline__ void write(O* h, float* gk, float* uk, uint32_t at, float sx, f32x4 gs, f32x4 us) const {
    float v[4], g[4], u[4], d;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      g[e] = sizeof(T) == 1 ? gs[e] * (sx * sg[e]) : gs[e] + bg[e];
      u[e] = sizeof(T) == 1 ? us[e] * (sx * su[e]) : us[e] + bu[e];
      v[e] = activate<ACT, false>(g[e], &d) * u[e];
    }
    store_n<O, 4>(h + at, v, WHOLE ? 4 : left);
    if (sizeof(T) > 1 && gk != nullptr) {
      store_n<float, 4>(gk + at, g, WHOLE ? 4 : left);
      store_n<float, 4>(uk + at, u, WHOLE ? 4 : left);
    }
  }
};

// WQ x WP waves, each JQ x JP blocks of 32 x 32.
//
// A step's operands are read while the step before it multiplies, across the slabs' ends too: the barrier that ends
// slab k (its last operands are in registers, slab k + 1 has landed) comes before k's last step, beside which k + 1's
// first operands are read and the rows of slab k + 2 are copied into the stage that k leaves. Columns have three
// stages: those of slab k + 2 are copied beside k's other steps and have a whole slab more to land.
template <typename T, typename O, bool QKM, bool PKM, bool GATED, int WQ, int WP, int JQ, int JP, int OCC>
__global__ __launch_bounds__(64 * WQ * WP, OCC) void gated_gemm_kernel(Params a) {
  constexpr int NW = WQ * WP, BQ = WQ * JQ * 32, BP = WP * JP * 32, QS = BQ * kSlab, PS = BP * kSlab;
  constexpr int STEPS = 4 / kCh<T>, MMAS = JQ * JP, READS = JQ + JP;
  static_assert(!GATED || JP % 2 == 0, "a wave holds gate blocks and the up blocks beside them");
  __shared__ __attribute__((aligned(1024))) char lds[2 * QS + 3 * PS];
  const Place at = place_of(a);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wq = w % WQ, wp = w / WQ;
  Copy<T, QKM, BQ, NW, false> cq;
  Copy<T, PKM, BP, NW, GATED> cp;
  constexpr int NQ = decltype(cq)::N, NP = decltype(cp)::N;
  Side q = a.q;
  if (at.turn > 0) q.b0 = a.q_turn;
  cq.init(q, (int64_t)at.q * BQ);
  cp.init(a.p, (int64_t)at.p * (GATED ? BP / 2 : BP));
  Read<T, QKM, BQ, JQ> rq;
  Read<T, PKM, BP, JP> rp;
  rq.init(wq * JQ);
  rp.init(wp * JP);
  f32x16 acc[JQ][JP];
#pragma unroll
  for (int i = 0; i < JQ; ++i)
#pragma unroll
    for (int j = 0; j < JP; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
  const int k0 = at.shared < 0 ? 0 : at.split * a.per_split, k_end = at.shared < 0 ? a.slabs : min(a.slabs, k0 + a.per_split);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds + w * 1024;
  typename Copy<T, QKM, BQ, NW, false>::Slab sq;
  typename Copy<T, PKM, BP, NW, GATED>::Slab sp;
  const auto prepare = [&](int k) {
    const int half = k >= a.half_slabs ? 1 : 0, kk = k - half * a.half_slabs;
    const int64_t left = k < k_end ? a.K - (int64_t)kk * (kSlab / (int)sizeof(T)) : 0;
    sq = cq.slab(half, kk, left);
    sp = cp.slab(half, kk, left);
  };
  Frag<T> fq[2][JQ], fp[2][JP];
  const auto read = [&](int set, int n, int s, int oq, int op) {
    if (n < JP) fp[set][n] = rp.get(lds + op, n, s);
    else fq[set][n - JP] = rq.get(lds + oq, n - JP, s);
  };
  // where the rows of slabs k and k + 1 lie, and the columns of k, k + 1 and k + 2
  int q0 = 0, q1 = QS, p0 = 2 * QS, p1 = p0 + PS, p2 = p1 + PS;
  const auto whole = [&](int k, int oq, int op) {
    prepare(k);
#pragma unroll
    for (int n = 0; n < NP; ++n) cp.issue(sp, n, lds0 + op);
#pragma unroll
    for (int n = 0; n < NQ; ++n) cq.issue(sq, n, lds0 + oq);
  };
  whole(k0, q0, p0);
  whole(k0 + 1, q1, p1);
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(NP + NQ) : "memory");
#pragma unroll
  for (int n = 0; n < READS; ++n) read(0, n, 0, q0, p0);
  for (int k = k0; k < k_end; ++k) {
    prepare(k + 2);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const bool last = s == STEPS - 1;
      // all but this slab's copies of columns have landed
      if (last) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(NP) : "memory");
#pragma unroll
      for (int n = 0; n < MMAS; ++n) {
        // next step's operands beside the first half of the products, and copies evenly
        constexpr int AT_ONCE = (2 * READS + MMAS - 1) / MMAS;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
          if (n * AT_ONCE + i < READS)
            read((s + 1) & 1, n * AT_ONCE + i, last ? 0 : s + 1, last ? q1 : q0, last ? p1 : p0);
        constexpr int EARLY = (STEPS - 1) * MMAS;
        const int m = s * MMAS + n;
#pragma unroll
        for (int i = 0; i < (NQ + MMAS - 1) / MMAS; ++i)
          if (last && n * NQ / MMAS + i < (n + 1) * NQ / MMAS) cq.issue(sq, n * NQ / MMAS + i, lds0 + q0);
#pragma unroll
        for (int i = 0; i < (NP + EARLY - 1) / EARLY; ++i)
          if (!last && m * NP / EARLY + i < (m + 1) * NP / EARLY) cp.issue(sp, m * NP / EARLY + i, lds0 + p2);
        mma(acc[n / JP][n % JP], fp[s & 1][n % JP], fq[s & 1][n / JP]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    const int t = p0;
    p0 = p1;
    p1 = p2;
    p2 = t;
    q1 = q0;
    q0 = QS - q0;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // zeros of slabs past the end: LDS is this workgroup's until then
  __syncthreads();
  // A wave's 32 rows at a time pass through LDS of its own, so that its lanes store whole runs of a row.
  constexpr int COLS = JP * 32, LD = COLS + 4, CPL = GATED ? 4 : 16 / (int)sizeof(O);
  constexpr int LPR = (GATED ? COLS / 2 : COLS) / CPL, ROWS = 64 / LPR;
  static_assert(NW * 32 * LD * 4 <= 2 * QS + 3 * PS, "fits the stages");
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
  float* mine = (float*)lds + w * 32 * LD;
  const int c = lane % LPR * CPL, r0 = lane / LPR;
  Columns<T, O> cols;
  if constexpr (GATED) cols.init(a, (int64_t)at.p * (BP / 2) + wp * (COLS / 2) + c);
  // Offsets within 32 rows fit 32 bits. A tile that lies inside the result needs no bounds.
  const int64_t rows0 = (int64_t)at.q * BQ + wq * JQ * 32, width = a.p.n;
  const bool inside = ((int64_t)at.q + 1) * BQ <= a.q.n && ((int64_t)at.p + 1) * (GATED ? BP / 2 : BP) <= width;
  const uint32_t step = ROWS * (uint32_t)width, first = r0 * (uint32_t)width + c;
#pragma unroll
  for (int i = 0; i < JQ; ++i) {
#pragma unroll
    for (int j = 0; j < JP; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *(f32x4*)(mine + l32 * LD + j * 32 + 8 * r + 4 * h) =
            f32x4{acc[i][j][4 * r], acc[i][j][4 * r + 1], acc[i][j][4 * r + 2], acc[i][j][4 * r + 3]};
    const int64_t row0 = rows0 + i * 32;
    if constexpr (GATED) {
      const int64_t to = row0 * width + (int64_t)at.p * (BP / 2) + wp * (COLS / 2);
      O* ph = (O*)a.h + to;
      float* pg = a.g != nullptr ? a.g + to : nullptr;
      float* pu = a.g != nullptr ? a.u + to : nullptr;
      const float* from = mine + (c >> 5) * 64 + (c & 31);
      const auto rows = [&](auto act, auto whole) {
#pragma unroll 4
        for (int r = 0; r < 32 / ROWS; ++r) {
          const int64_t row = row0 + r0 + r * ROWS;
          if (!decltype(whole)::value && (row >= a.q.n || cols.left <= 0)) continue;
          const float* v = from + (r0 + r * ROWS) * LD;
          cols.template write<decltype(act)::value, decltype(whole)::value>(ph, pg, pu, first + r * step,
                                                                            sizeof(T) == 1 ? a.sx[row] : 1.0f, *(const f32x4*)v,
                                                                            *(const f32x4*)(v + 32));
        }
      };
      with_activation(a.act, [&](auto act) { inside ? rows(act, std::true_type()) : rows(act, std::false_type()); });
    } else {
      const int64_t left = width - ((int64_t)at.p * BP + wp * COLS + c);
      const int64_t to = row0 * width + (int64_t)at.p * BP + wp * COLS;
      O* out = (O*)a.out[at.turn] + to;
      float* part = a.part + (((int64_t)at.shared * a.splits + at.split) * BQ + (wq * JQ + i) * 32) * BP + wp * COLS;
      const auto rows = [&](auto* out, uint32_t first, uint32_t step, auto whole) {
        typedef std::remove_pointer_t<decltype(out)> R;
#pragma unroll 4
        for (int r = 0; r < 32 / ROWS; ++r) {
          if (!decltype(whole)::value && (row0 + r0 + r * ROWS >= a.q.n || left <= 0)) continue;
          float v[CPL];
#pragma unroll
          for (int e = 0; e < CPL; e += 4) *(f32x4*)(v + e) = *(const f32x4*)(mine + (r0 + r * ROWS) * LD + c + e);
          store_n<R, CPL>(out + first + r * step, v, decltype(whole)::value ? CPL : left);
        }
      };
      if (at.shared >= 0) rows(part, r0 * BP + c, ROWS * BP, std::true_type());
      else if (inside) rows(out, first, step, std::true_type());
      else rows(out, first, step, std::false_type());
    }
  }
}

// ---- few rows -----------------------------------------------------------------------------
// Up to 64 rows: bound by reading the weights. A workgroup has 16 gate and 16 up rows; its four waves share the inner
// dimension, each with its operands straight from memory into registers, a slab of 128 bytes ahead, and their
// sums are added in wave order in LDS. A slab's loads are issued together: each takes 16 rows' lines in part, and
// those that follow find them on their way. What is in flight has to fit the L1, or lines are fetched again. Four rows,
// D = 4096, F = 11264, bf16, one, two and three slabs ahead: 36.1, 38.6 and 61.4 us (5.1 TB/s, as a copy); eight waves and
// one slab 38.4; 32 columns a workgroup by 32-wide products with four steps of 32 bytes ahead 70.
constexpr int kFewWaves = 4;
constexpr int kFewCols = 16;

// 16 x 16 results: lane l holds row (column) l % 16 and, of each 64 bytes of the inner dimension, quarter l / 16 (8 bits:
// of each 128).
__device__ __forceinline__ void mma16(f32x4& d, const Frag<bf16>& a, const Frag<bf16>& b) {
  d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.c[0]), __builtin_bit_cast(bf16x8, b.c[0]), d, 0, 0, 0);
}
__device__ __forceinline__ void mma16(f32x4& d, const Frag<f16>& a, const Frag<f16>& b) {
  d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.c[0]), __builtin_bit_cast(f16x8, b.c[0]), d, 0, 0, 0);
}
__device__ __forceinline__ void mma16(f32x4& d, const Frag<float>& a, const Frag<float>& b) {
  const f32x4 x = __builtin_bit_cast(f32x4, a.c[0]), y = __builtin_bit_cast(f32x4, b.c[0]);
#pragma unroll
  for (int e = 0; e < 4; ++e) d = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], d, 0, 0, 0);
}
__device__ __forceinline__ void mma16(f32x4& d, const Frag<e4m3>& a, const Frag<e4m3>& b) {
  d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(a), wide(b), d, 0, 0, 0, 0, 0, 0);
}

template <typename T, typename O, int JQ>
__global__ __launch_bounds__(64 * kFewWaves, 2) void gated_few_kernel(Params a) {
  constexpr int STEPS = 2 / kCh<T>, E = sizeof(T);  // of a slab
  __shared__ float sums[kFewWaves][JQ][2][4][64];
  const int lane = threadIdx.x & 63, l16 = lane & 15, quarter = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t f0 = (int64_t)blockIdx.x * kFewCols, f = min(f0 + l16, a.p.n - 1);
  const char* wg = a.p.b0 + f * a.p.ld;
  const char* wu = a.p.b1 + f * a.p.ld;
  const char* x[JQ];
#pragma unroll
  for (int i = 0; i < JQ; ++i) x[i] = a.q.b0 + min((int64_t)(i * 16 + l16), a.q.n - 1) * a.q.ld;
  const int64_t row = a.K * E;  // bytes
  const int slabs = (int)cdiv(row, kSlab), per = (slabs + kFewWaves - 1) / kFewWaves, s0 = w * per, s1 = min(slabs, s0 + per);
  f32x4 ag[JQ], au[JQ];
#pragma unroll
  for (int i = 0; i < JQ; ++i) ag[i] = au[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  Frag<T> fg[STEPS], fu[STEPS], fx[STEPS][JQ];
  const auto load = [&](int s) {
#pragma unroll
    for (int t = 0; t < STEPS; ++t)
#pragma unroll
      for (int c = 0; c < kCh<T>; ++c) {
        const int64_t at = (int64_t)s * kSlab + (kCh<T> == 1 ? t * 64 + quarter * 16 : quarter * 32 + c * 16);
        const bool in = s < s1 && at < row;
        const int64_t o = in ? at : 0;
        const u32x4 zero = {0, 0, 0, 0}, vg = *(const u32x4*)(wg + o), vu = *(const u32x4*)(wu + o);
        fg[t].c[c] = in ? vg : zero;
        fu[t].c[c] = in ? vu : zero;
#pragma unroll
        for (int i = 0; i < JQ; ++i) {
          const u32x4 vx = *(const u32x4*)(x[i] + o);
          fx[t][i].c[c] = in ? vx : zero;
        }
      }
  };
  load(s0);
  for (int s = s0; s < s1; ++s) {
    Frag<T> g[STEPS], u[STEPS], v[STEPS][JQ];
#pragma unroll
    for (int t = 0; t < STEPS; ++t) {
      g[t] = fg[t];
      u[t] = fu[t];
#pragma unroll
      for (int i = 0; i < JQ; ++i) v[t][i] = fx[t][i];
    }
    load(s + 1);
#pragma unroll
    for (int t = 0; t < STEPS; ++t)
#pragma unroll
      for (int i = 0; i < JQ; ++i) {
        mma16(ag[i], g[t], v[t][i]);
        mma16(au[i], u[t], v[t][i]);
      }
  }
#pragma unroll
  for (int i = 0; i < JQ; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sums[w][i][0][e][lane] = ag[i][e];
      sums[w][i][1][e][lane] = au[i][e];
    }
  __syncthreads();
  if (w >= JQ) return;  // wave w ends block w
  f32x4 g, u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    g[e] = u[e] = 0.0f;
#pragma unroll
    for (int v = 0; v < kFewWaves; ++v) {
      g[e] += sums[v][w][0][e][lane];
      u[e] += sums[v][w][1][e][lane];
    }
  }
  Columns<T, O> cols;
  cols.init(a, f0 + 4 * quarter);
  const int64_t m = w * 16 + l16;
  if (m >= a.q.n || cols.left <= 0) return;
  const uint32_t to = (uint32_t)(m * a.p.n + cols.col);  // 64 rows of up to 2^20
  const float sx = sizeof(T) == 1 ? a.sx[m] : 1.0f;
  with_activation(a.act, [&](auto act) {
    cols.template write<decltype(act)::value, false>((O*)a.h, a.g, a.u, to, sx, g, u);
  });
}

// ---- dg and du ----------------------------------------------------------------------------
constexpr int kActThreads = 256;
constexpr int kActCols = 4;  // columns of a thread

// dg and du [M, ld], zeros past F, and with `part` the column sums of a workgroup's rows, before their rounding.
template <typename T, int ACT>
__global__ __launch_bounds__(kActThreads) void gated_act_bwd_kernel(const T* __restrict__ dh, const float* __restrict__ g,
                                                                    const float* __restrict__ u, T* __restrict__ dg,
                                                                    T* __restrict__ du, float* __restrict__ part, int64_t M,
                                                                    int64_t F, int64_t ld, int rows, int strips) {
  const int strip = blockIdx.x % strips;
  const int64_t blk = blockIdx.x / strips, col = ((int64_t)strip * kActThreads + threadIdx.x) * kActCols;
  const int64_t r0 = blk * rows, r1 = min(M, r0 + rows);
  if (col >= ld) return;
  const int n = (int)max((int64_t)0, min((int64_t)kActCols, F - col));
  float sg[kActCols] = {}, su[kActCols] = {};
#pragma unroll 2
  for (int64_t r = r0; r < r1; ++r) {
    float vd[kActCols], vg[kActCols], vu[kActCols], og[kActCols], ou[kActCols];
    const int64_t at = r * F + col;
    if (n == kActCols) {
      const vec_t<T, 4> d = load_any<T, 4>(dh + at);
      const vec_t<float, 4> a = load_any<float, 4>(g + at), b = load_any<float, 4>(u + at);
#pragma unroll
      for (int e = 0; e < kActCols; ++e) vd[e] = to_f32(d[e]), vg[e] = a[e], vu[e] = b[e];
    } else {
#pragma unroll
      for (int e = 0; e < kActCols; ++e) {
        vd[e] = e < n ? to_f32(dh[at + e]) : 0.0f;
        vg[e] = e < n ? g[at + e] : 0.0f;
        vu[e] = e < n ? u[at + e] : 0.0f;
      }
    }
#pragma unroll
    for (int e = 0; e < kActCols; ++e) {
      float d;
      const float a = activate<ACT, true>(vg[e], &d);
      og[e] = vd[e] * vu[e] * d;
      ou[e] = vd[e] * a;
      if (part != nullptr) {
        sg[e] += og[e];
        su[e] += ou[e];
      }
    }
    store_n<T, 4>(dg + r * ld + col, og, ld - col);
    store_n<T, 4>(du + r * ld + col, ou, ld - col);
  }
  if (part == nullptr) return;
#pragma unroll
  for (int e = 0; e < kActCols; ++e) {
    if (e >= n) break;
    part[blk * 2 * F + col + e] = sg[e];
    part[blk * 2 * F + F + col + e] = su[e];
  }
}

// The shared tiles' sums added in the splits' order: 1024 elements of a tile a workgroup, four splits' loads in flight.
template <typename O> __global__ __launch_bounds__(256) void gated_join_kernel(Params a, int B) {
  const int per = B * B / 1024, tile = blockIdx.x / per, at = (blockIdx.x % per) * 1024 + threadIdx.x * 4;
  const Place t = tile_of(a, a.whole + tile);
  const int64_t row = (int64_t)t.q * B + at / B, col = (int64_t)t.p * B + at % B;
  if (row >= a.q.n || col >= a.p.n) return;
  const float* from = a.part + (int64_t)tile * a.splits * B * B + at;
  float v[4] = {};
#pragma unroll 4
  for (int k = 0; k < a.splits; ++k) {
    const f32x4 p = *(const f32x4*)(from + (int64_t)k * B * B);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += p[e];
  }
  store_n<O, 4>((O*)a.out[t.turn] + row * a.p.n + col, v, a.p.n - col);
}

// ---- launches -----------------------------------------------------------------------------
constexpr int kCus = 256;
// Rows that the kernel for few of them takes: 64, or 32 where the weights are large. bf16, its times and the tiles':
// D = 4096, F = 11264: 32 rows 55 and 54 us, 64 rows 76 and 54; D = 1024, F = 4096: 64 rows 9.7 and 12.2.
constexpr int64_t kFewRows = 64, kFewRowsLarge = 32, kLargeWeight = 1 << 23;
constexpr int kBiasBlocks = 256;

struct Split {
  bool small;
  int tq, tp, whole, splits, per_split, slabs;
  int64_t shared;  // tiles that are cut
  size_t part_bytes() const { return (size_t)(shared * splits) * (small ? 128 * 128 : 256 * 256) * 4; }
};

// The tile, and into how many parts the inner dimension of the tiles is cut that do not fill the CUs a last time (for
// few tiles, all of them): what an estimate of the time says. A CU holds one workgroup of 256 x 256 or two of 128 x 128.
// Microseconds a slab and a tile's start and end, as measured:
//               256 x 256, on every CU   on some   128 x 128, two on a CU   one
//     16 bits   1.45                     1.3       0.9                      0.5
//     fp32      7.3                      7.3       3.6                      1.95
//     around    10                                 6
// `around` is silu's, without g and u: a tile of 256 x 256 with gelu takes about 14 around, and the forward of 8192 x 768 x
// 2048 with both 73 us where this says 55. A join writes and reads 6 MB a microsecond; what is split has to promise 3% more
// than that. bf16, dx of 8192 x 768 x 2048: tiles of 256 80 us, in two parts 72; of 128 59, in two parts 80. dx of 5000 x
// 1024 x 3000: 113 and in three parts 80; 94 and 93. dx of 300 x 768 x 2048: of 128 31, in four parts 14. dx of 8192 x 4096
// x 11264: 1098 and 1485; its dW, 1408 tiles of 256, 1218, the last 128 in two parts 1183.
Split split_of(int64_t rows, int64_t cols, int64_t turns, int64_t slabs, int64_t es, bool may_split) {
  Split best = {};
  double least = -1.0;
  for (int small = 0; small < 2; ++small) {
    const int64_t b = small ? 128 : 256, slots = small ? 2 * kCus : kCus, tq = cdiv(rows, b), tp = cdiv(cols, b);
    const int64_t tiles = tq * tp * turns, rest = tiles % slots;
    const double around = small ? 6.0 : 10.0, all = es == 4 ? (small ? 3.6 : 7.3) : (small ? 0.9 : 1.45);
    const double some = es == 4 ? (small ? 1.95 : 7.3) : (small ? 0.5 : 1.3);
    const double full = (double)(tiles / slots) * ((double)slabs * all + around);
    for (int64_t n = 1; n <= 16; ++n) {
      const int64_t per = cdiv(slabs, n), groups = rest * n;
      if (n > 1 && (!may_split || rest == 0 || slabs < 4 * n || cdiv(slabs, per) != n || groups > 2 * slots)) continue;
      double time = full;
      if (rest > 0)
        time += (double)cdiv(groups, slots) * ((double)per * (groups < kCus || (small && groups == kCus) ? some : all) + around);
      if (n > 1) time += 3.0 + 0.03 * time + (double)(rest * b * b) * (8.0 * (double)n + 2.0) / 6e6;
      if (least < 0.0 || time < least) {
        least = time;
        best = Split{small != 0, (int)tq, (int)tp, (int)(n > 1 ? tiles - rest : tiles), (int)n, (int)per, (int)slabs, n > 1 ? rest : 0};
      }
    }
  }
  return best;
}

template <typename T, typename O, bool QKM, bool PKM, bool GATED> int gemm(Params p, const Split& s, hipStream_t st) {
  p.tq = s.tq;
  p.tp = s.tp;
  p.whole = s.whole;
  p.splits = s.splits;
  p.per_split = s.per_split;
  p.slabs = s.slabs;
  const unsigned grid = (unsigned)(s.whole + s.shared * s.splits);
  if (grid == 0) return SPARTON_OK;
  if (s.small)
    hipLaunchKernelGGL((gated_gemm_kernel<T, O, QKM, PKM, GATED, 2, 2, 2, 2, 2>), dim3(grid), dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((gated_gemm_kernel<T, O, QKM, PKM, GATED, 2, 2, 4, 4, 1>), dim3(grid), dim3(256), 0, st, p);
  if (s.shared > 0) {
    const int B = s.small ? 128 : 256;
    hipLaunchKernelGGL(gated_join_kernel<O>, dim3((unsigned)(s.shared * (B * B / 1024))), dim3(256), 0, st, p, B);
  }
  return (int)hipGetLastError();
}

int64_t es_of(int dtype) { return dtype == SPARTON_F32 ? 4 : 2; }
int64_t pad_of(int64_t F, int dtype) { return round_up(F, 16 / es_of(dtype)); }

int check(int64_t M, int64_t D, int64_t F, int dtype, int64_t es, int act) {
  if (M < 0 || D <= 0 || F < 0 || dtype < SPARTON_F32 || dtype > SPARTON_F16) return SPARTON_EINVAL;
  if (act < SPARTON_SILU || act > SPARTON_RELU || D * es % 16 != 0) return SPARTON_EINVAL;
  // 256 rows of an operand lie within 2^31 bytes
  if (D > (1 << 20) || F > (1 << 20) || M > INT32_MAX) return SPARTON_EUNSUPPORTED;
  const uint64_t tiles = std::max((uint64_t)cdiv(std::max<int64_t>(M, 1), 128) * cdiv(std::max(F, D), 64),
                                  (uint64_t)cdiv(F, 128) * cdiv(D, 128) * 2);
  return tiles * 256 >= kMaxThreads ? SPARTON_EUNSUPPORTED : SPARTON_OK;
}

template <typename T, typename O> int forward(Params& p, hipStream_t st) {
  p.turns = 1;
  if (p.q.n <= (p.p.n * p.K > kLargeWeight ? kFewRowsLarge : kFewRows)) {
    const dim3 grid((unsigned)cdiv(p.p.n, kFewCols)), block(64 * kFewWaves);
    if (p.q.n <= 16) hipLaunchKernelGGL((gated_few_kernel<T, O, 1>), grid, block, 0, st, p);
    else if (p.q.n <= 32) hipLaunchKernelGGL((gated_few_kernel<T, O, 2>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((gated_few_kernel<T, O, 4>), grid, block, 0, st, p);
    return (int)hipGetLastError();
  }
  const int64_t slabs = cdiv(p.K * (int64_t)sizeof(T), kSlab);
  p.half_slabs = (int)slabs;
  return gemm<T, O, false, false, true>(p, split_of(p.q.n, 2 * p.p.n, 1, slabs, sizeof(T), false), st);
}

struct Plan {
  Split dx, dw;
  size_t act, part, bias;  // bytes
  int rows, strips, blocks;
};

Plan plan_of(int64_t M, int64_t D, int64_t F, int dtype, bool with_bias) {
  const int64_t es = es_of(dtype), ld = pad_of(F, dtype);
  Plan p;
  p.dx = split_of(M, D, 1, 2 * cdiv(F * es, kSlab), es, true);
  p.dw = split_of(F, D, 2, cdiv(M * es, kSlab), es, true);
  p.act = (size_t)round_up(2 * M * ld * es, 256);
  p.part = std::max(p.dx.part_bytes(), p.dw.part_bytes());  // of whole 256 bytes
  p.strips = (int)cdiv(ld, kActThreads * kActCols);
  const int64_t want = with_bias ? kBiasBlocks : 4096;
  p.rows = (int)std::max<int64_t>(1, cdiv(M * (with_bias ? 1 : p.strips), want));
  p.blocks = (int)cdiv(M, p.rows);
  p.bias = with_bias ? (size_t)round_up((int64_t)p.blocks * 2 * F * 4, 256) : 0;
  return p;
}

template <typename T>
int backward(const T* dh, const char* x, const char* wg, const char* wu, const float* g, const float* u, T* dx, T* dwg, T* dwu,
             T* dbg, T* dbu, char* ws, int64_t M, int64_t D, int64_t F, int act, int dtype, hipStream_t st) {
  constexpr int64_t E = sizeof(T);
  const bool with_bias = dbg != nullptr || dbu != nullptr;
  const Plan pl = plan_of(M, D, F, dtype, with_bias);
  const int64_t ld = pad_of(F, dtype);
  T* dg = (T*)ws;
  T* du = dg + M * ld;
  float* part = (float*)(ws + pl.act);
  float* bias = with_bias ? (float*)(ws + pl.act + pl.part) : nullptr;
  if (M > 0) {
    const auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)(pl.blocks * (int64_t)pl.strips)), dim3(kActThreads), 0, st, dh, g, u, dg, du, bias,
                         M, F, ld, pl.rows, pl.strips);
    };
    if (act == SPARTON_SILU) launch(gated_act_bwd_kernel<T, SPARTON_SILU>);
    else if (act == SPARTON_GELU) launch(gated_act_bwd_kernel<T, SPARTON_GELU>);
    else if (act == SPARTON_GELU_TANH) launch(gated_act_bwd_kernel<T, SPARTON_GELU_TANH>);
    else launch(gated_act_bwd_kernel<T, SPARTON_RELU>);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  if (with_bias) {
    hipLaunchKernelGGL(colsum_kernel, dim3((unsigned)cdiv(2 * F, 64)), dim3(64 * kSumWaves), 0, st, (const float*)bias,
                       M > 0 ? pl.blocks : 0, (int)F, (int)(2 * F), dbg, dbu, dtype);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  if (dx != nullptr && M > 0) {
    Params p = {};
    p.q = Side{(const char*)dg, (const char*)du, ld * E, M};
    p.p = Side{wg, wu, D * E, D};
    p.K = F;
    p.half_slabs = (int)cdiv(F * E, kSlab);
    p.turns = 1;
    p.out[0] = dx;
    p.part = part;
    const int rc = gemm<T, T, false, true, false>(p, pl.dx, st);
    if (rc != 0) return rc;
  }
  if (dwg != nullptr) {
    Params p = {};
    p.q = Side{(const char*)dg, (const char*)dg, ld * E, F};
    p.q_turn = (const char*)du;
    p.p = Side{x, x, D * E, D};
    p.K = M;
    p.half_slabs = (int)cdiv(M * E, kSlab);
    p.turns = 2;
    p.out[0] = dwg;
    p.out[1] = dwu;
    p.part = part;
    const int rc = gemm<T, T, true, true, false>(p, pl.dw, st);
    if (rc != 0) return rc;
  }
  return SPARTON_OK;
}

}  // namespace gated
}  // namespace sparton

using namespace sparton;

#define SPARTON_EXPORT extern "C" __attribute__((visibility("default")))

SPARTON_EXPORT int sparton_gated_fwd(const void* x, const void* w_gate, const void* w_up, const void* b_gate, const void* b_up,
                                     int activation, void* h, float* gate, float* up, int64_t M, int64_t D, int64_t F, int dtype,
                                     void* stream) {
  const int rc = gated::check(M, D, F, dtype, dtype == SPARTON_F32 ? 4 : 2, activation);
  if (rc != SPARTON_OK) return rc;
  if (M == 0 || F == 0) return SPARTON_OK;
  if (x == nullptr || w_gate == nullptr || w_up == nullptr || h == nullptr || (gate == nullptr) != (up == nullptr))
    return SPARTON_EINVAL;
  const uintptr_t es = (uintptr_t)gated::es_of(dtype);
  if (!aligned(x, 16) || !aligned(w_gate, 16) || !aligned(w_up, 16) || !aligned(h, es) || !aligned(b_gate, es) ||
      !aligned(b_up, es) || !aligned(gate, 4) || !aligned(up, 4))
    return SPARTON_EALIGN;
  gated::Params p = {};
  p.q = gated::Side{(const char*)x, (const char*)x, D * (int64_t)es, M};
  p.p = gated::Side{(const char*)w_gate, (const char*)w_up, D * (int64_t)es, F};
  p.K = D;
  p.h = h;
  p.g = gate;
  p.u = up;
  p.bg = b_gate;
  p.bu = b_up;
  p.act = activation;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SPARTON_BF16) return gated::forward<bf16, bf16>(p, st);
  if (dtype == SPARTON_F16) return gated::forward<f16, f16>(p, st);
  return gated::forward<float, float>(p, st);
}

SPARTON_EXPORT int sparton_gated_fwd_quantized(const void* x, const float* x_scale, const void* w_gate, const float* gate_scale,
                                          const void* w_up, const float* up_scale, int activation, void* h, int64_t M,
                                          int64_t D, int64_t F, int out_dtype, void* stream) {
  const int rc = gated::check(M, D, F, out_dtype, 1, activation);
  if (rc != SPARTON_OK) return rc;
  if (M == 0 || F == 0) return SPARTON_OK;
  if (x == nullptr || w_gate == nullptr || w_up == nullptr || h == nullptr || x_scale == nullptr || gate_scale == nullptr ||
      up_scale == nullptr)
    return SPARTON_EINVAL;
  if (!aligned(x, 16) || !aligned(w_gate, 16) || !aligned(w_up, 16) || !aligned(h, (uintptr_t)gated::es_of(out_dtype)) ||
      !aligned(x_scale, 4) || !aligned(gate_scale, 4) || !aligned(up_scale, 4))
    return SPARTON_EALIGN;
  gated::Params p = {};
  p.q = gated::Side{(const char*)x, (const char*)x, D, M};
  p.p = gated::Side{(const char*)w_gate, (const char*)w_up, D, F};
  p.K = D;
  p.h = h;
  p.sx = x_scale;
  p.sg = gate_scale;
  p.su = up_scale;
  p.act = activation;
  hipStream_t st = (hipStream_t)stream;
  if (out_dtype == SPARTON_BF16) return gated::forward<gated::e4m3, bf16>(p, st);
  if (out_dtype == SPARTON_F16) return gated::forward<gated::e4m3, f16>(p, st);
  return gated::forward<gated::e4m3, float>(p, st);
}

SPARTON_EXPORT size_t sparton_gated_workspace_bytes(int64_t M, int64_t D, int64_t F, int with_bias, int dtype) {
  if (gated::check(M, D, F, dtype, dtype == SPARTON_F32 ? 4 : 2, SPARTON_SILU) != SPARTON_OK || M == 0 || F == 0) return 0;
  const gated::Plan p = gated::plan_of(M, D, F, dtype, with_bias != 0);
  return p.act + p.part + p.bias;
}

SPARTON_EXPORT int sparton_gated_bwd(const void* dh, const void* x, const void* w_gate, const void* w_up, const float* gate,
                                     const float* up, int activation, void* dx, void* d_w_gate, void* d_w_up, void* d_b_gate,
                                     void* d_b_up, void* workspace, size_t workspace_bytes, int64_t M, int64_t D, int64_t F,
                                     int dtype, void* stream) {
  const int rc = gated::check(M, D, F, dtype, dtype == SPARTON_F32 ? 4 : 2, activation);
  if (rc != SPARTON_OK) return rc;
  if ((d_w_gate == nullptr) != (d_w_up == nullptr)) return SPARTON_EINVAL;
  if (F == 0 && (dx != nullptr || d_w_gate != nullptr)) return SPARTON_EUNSUPPORTED;
  if (F == 0) return SPARTON_OK;
  if (M > 0 && (dh == nullptr || x == nullptr || w_gate == nullptr || w_up == nullptr || gate == nullptr || up == nullptr))
    return SPARTON_EINVAL;
  const uintptr_t es = (uintptr_t)gated::es_of(dtype);
  if (!aligned(x, 16) || !aligned(w_gate, 16) || !aligned(w_up, 16) || !aligned(dh, es) || !aligned(dx, es) ||
      !aligned(d_w_gate, es) || !aligned(d_w_up, es) || !aligned(d_b_gate, es) || !aligned(d_b_up, es) || !aligned(gate, 4) ||
      !aligned(up, 4))
    return SPARTON_EALIGN;
  const bool with_bias = d_b_gate != nullptr || d_b_up != nullptr;
  const size_t need = sparton_gated_workspace_bytes(M, D, F, with_bias, dtype);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return SPARTON_EWORKSPACE;
  if (need > 0 && !aligned(workspace, 256)) return SPARTON_EALIGN;
  hipStream_t st = (hipStream_t)stream;
  const char *cx = (const char*)x, *cg = (const char*)w_gate, *cu = (const char*)w_up;
  char* ws = (char*)workspace;
  if (dtype == SPARTON_BF16)
    return gated::backward<bf16>((const bf16*)dh, cx, cg, cu, gate, up, (bf16*)dx, (bf16*)d_w_gate, (bf16*)d_w_up, (bf16*)d_b_gate,
                                 (bf16*)d_b_up, ws, M, D, F, activation, dtype, st);
  if (dtype == SPARTON_F16)
    return gated::backward<f16>((const f16*)dh, cx, cg, cu, gate, up, (f16*)dx, (f16*)d_w_gate, (f16*)d_w_up, (f16*)d_b_gate,
                                (f16*)d_b_up, ws, M, D, F, activation, dtype, st);
  return gated::backward<float>((const float*)dh, cx, cg, cu, gate, up, (float*)dx, (float*)d_w_gate, (float*)d_w_up,
                                (float*)d_b_gate, (float*)d_b_up, ws, M, D, F, activation, dtype, st);
}
