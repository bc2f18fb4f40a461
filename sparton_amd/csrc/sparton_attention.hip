// Attention of a backbone layer, forward and backward, on gfx950:
//     s_ij = scale q_i . k_j            over the keys j that row i may look at
//     p_ij = exp(s_ij - L_i),  L_i = log sum_j exp(s_ij),   o_i = sum_j p_ij v_j
//     delta_i = do_i . o_i,   ds_ij = p_ij (do_i . v_j - delta_i)
//     dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
// A key takes part where the key mask is nonzero and, with `causal`, where j <= i + Sk - Sq. Query
// head h reads key head h / (Hq / Hk); dk and dv are summed over the heads that share one. A row with
// no key gives o = 0 and zero gradients. Keys that take no part are never multiplied: what their
// memory holds (NaN, infinities) reaches no output.
//
// Every product runs on 32x32 MFMAs with fp32 sums, in transposed form: a wave holds 32 rows as the
// columns of its results, one column per lane (and per half of the wave half of that column's
// values). Row statistics are then lane scalars, and the probabilities lie in registers as the next
// product's right operand: lane l holds, of its column, the inner indices 8 q + 4 (l / 32) + e, and
// the left operand is read from LDS in that order. Nothing is exchanged between lanes but the two
// halves' maxima and sums.

#include <math.h>

#include <algorithm>

#include "sparton_common.h"

namespace sparton {
namespace attn {

constexpr float kLog2e = 1.44269504088896341f;
constexpr int kThreads = 256;
constexpr int kMaxSplits = 64;  // the combining wave holds one split's weight per lane

typedef __attribute__((ext_vector_type(4))) short s16x4;

struct Strides {
  int64_t b, h, s;
};

struct Params {
  const void *q, *k, *v, *mask, *o, *dout;
  void *out, *dq, *dk, *dv;
  float *lse, *delta;      // [B, Hq, Sq]: log2 of the row sums; do . o
  float *part, *part_lse;  // partial outputs of a split over keys: [B, Hk, splits, R, D] and [B, Hk, splits, R]
  Strides sq, sk, sv, so, sdo, sdq, sdk, sdv;
  int64_t mask_b;
  int B, Hq, Hk, G, Sq, Sk, D, R;  // G query heads share a key head; R = G Sq rows look at one key head
  int mask_dtype, causal, splits, tiles_per_split;
  float scale, c;  // c = scale log2(e)
};

// ---- geometry of one head dimension and type ---------------------------------------------
// An operand fragment is 16 bytes per lane: eight 16-bit or four fp32 values along the inner index.
// KC inner indices make one step (two 16-byte chunks, one per half of the wave).
template <typename T, int DH> struct Geo {
  static constexpr int ES = sizeof(T);
  static constexpr int EPC = 16 / ES;       // elements of a 16-byte chunk
  static constexpr int KC = 2 * EPC;        // inner indices of a step
  static constexpr int NC = DH / KC;        // steps along the head dimension
  static constexpr int PB = 32 / KC;        // steps along 32 rows
  static constexpr int ROW = DH * ES;       // bytes of an LDS row
  static constexpr int CPR = DH * ES / 16;  // chunks of a row
  static constexpr int DB = DH / 32;        // 32-row blocks of a transposed output
};

// LDS rows are ROW bytes; the chunks of row r are permuted by XOR with f(r), so that the 32 lanes
// that read one chunk of 32 rows spread over all banks.
template <int ROW, int CPR> __device__ __forceinline__ int swz(int r) {
  constexpr int SH = ROW >= 128 ? 0 : ROW >= 64 ? 1 : 2;
  constexpr int MASK = (CPR < 16 ? CPR : 16) - 1;
  return (r >> SH) & MASK;
}
template <typename T, int DH> __device__ __forceinline__ int lds_at(int row, int chunk) {
  typedef Geo<T, DH> Gm;
  return row * Gm::ROW + ((chunk ^ swz<Gm::ROW, Gm::CPR>(row)) << 4);
}

template <typename T> struct Frag;
template <> struct Frag<bf16> { typedef bf16x8 type; };
template <> struct Frag<f16> { typedef f16x8 type; };
template <> struct Frag<float> { typedef f32x4 type; };
template <typename T> using frag_t = typename Frag<T>::type;

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// fp32: the step's inner index 2 takes element e of both halves, four times.
__device__ __forceinline__ f32x16 mma(f32x4 a, f32x4 b, f32x16 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

template <typename T> __device__ __forceinline__ frag_t<T> lds_frag(const char* p) { return *(const frag_t<T>*)p; }

// Left operand of a product over rows: element e of lane l is row0 + rho(l, e), column 32 db + l % 32,
// with rho the order in which a result's registers hold their rows. 16-bit: two transposing reads,
// each of which gives a lane four rows of its column; fp32: four plain reads.
template <typename T, int DH>
__device__ __forceinline__ frag_t<T> lds_cols(const char* tile, int row0, int db, int lane) {
  if constexpr (sizeof(T) == 2) {
    const int q = lane & 15;
    const int d = db * 32 + ((lane >> 4) & 1) * 16 + (q & 3) * 4;
    const int r = row0 + (lane >> 5) * 4 + (q >> 2);
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(tile + lds_at<T, DH>(r, d >> 3) + (d & 7) * 2));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(tile + lds_at<T, DH>(r + 8, d >> 3) + (d & 7) * 2));
    return __builtin_bit_cast(frag_t<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    const int d = db * 32 + (lane & 31);
    frag_t<T> f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = row0 + (lane >> 5) * 4 + e;
      f[e] = *(const float*)(tile + lds_at<T, DH>(r, d >> 2) + (d & 3) * 4);
    }
    return f;
  }
}

// Registers [KC/2 c, KC/2 (c + 1)) of a result as the right operand of step c, rounded to T. The
// rounding of a probability (or of ds) to 16 bits is off by at most half a step of its own value,
// and independent from key to key: it adds to an output's error what the output's own rounding does.
template <typename T> __device__ __forceinline__ frag_t<T> pack(const f32x16& s, int c) {
  constexpr int N = 16 / sizeof(T);
  frag_t<T> f;
#pragma unroll
  for (int e = 0; e < N; ++e) f[e] = from_f32<T>(s[c * N + e]);
  return f;
}

// Row of register r within a 32-row result block, before the half's 4.
__device__ __forceinline__ constexpr int reg_row(int r) { return 8 * (r / 4) + r % 4; }

__device__ __forceinline__ float other_half_max(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x),
                                                  false, false);
  return fmaxf(__builtin_bit_cast(float, (unsigned)s[0]), __builtin_bit_cast(float, (unsigned)s[1]));
}
__device__ __forceinline__ float other_half_sum(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x),
                                                  false, false);
  return __builtin_bit_cast(float, (unsigned)s[0]) + __builtin_bit_cast(float, (unsigned)s[1]);
}

// Consecutive workgroups go to the eight XCDs in turn; this numbering gives each XCD a contiguous
// range instead, so that the tiles of one head share their keys and values in that XCD's L2.
__device__ __forceinline__ int xcd_range(int w, int n) {
  const int x = w & 7, base = n >> 3, rem = n & 7;
  return x * base + min(x, rem) + (w >> 3);
}

__device__ __forceinline__ bool key_on(const void* mask, int mask_dtype, int64_t off) {
  switch (mask_dtype) {  // uniform
    case SPARTON_MASK_I64: return ((const int64_t*)mask)[off] != 0;
    case SPARTON_MASK_I32: return ((const int32_t*)mask)[off] != 0;
    default: return ((const uint8_t*)mask)[off] != 0;
  }
}

// The key mask of one batch row as bits, 64 words of 32 keys at a time, one word per lane. Every wave
// keeps its own copy; a word is read back as a scalar, so that a tile without keys costs a branch.
struct KeyBits {
  const void* mask;
  int64_t row;
  int dtype, kend, chunk;
  uint32_t word;
  __device__ __forceinline__ void init(const Params& p, int b, int kend_) {
    mask = p.mask;
    row = (int64_t)b * p.mask_b;
    dtype = p.mask_dtype;
    kend = kend_;
    chunk = -1;
    word = 0;
  }
  __device__ __forceinline__ void load(int c) {  // keys [2048 c, 2048 (c + 1))
    const int lane = threadIdx.x & 63;
    const int k0 = c * 2048;
    const int n = min(32, (kend - k0 + 63) >> 6);
    chunk = c;
    word = 0;
    for (int x = 0; x < n; ++x) {
      const int key = k0 + x * 64 + lane;
      bool on = key < kend;
      if (mask != nullptr) on = key_on(mask, dtype, row + min(key, kend - 1)) && on;
      const uint64_t bits = __ballot(on);
      word = lane == 2 * x ? (uint32_t)bits : lane == 2 * x + 1 ? (uint32_t)(bits >> 32) : word;
    }
  }
  // word of keys [32 blk, 32 blk + 32); blk < cdiv(kend, 32) rounded up to a tile
  __device__ __forceinline__ uint32_t at(int blk) {
    return (uint32_t)__builtin_amdgcn_readlane((int)word, blk & 63);
  }
  // The first tile after t, below t_end, of NW words, that has a key: its words in w.
  template <int NW> __device__ __forceinline__ int next(int t, int t_end, uint32_t (&w)[NW]) {
    for (++t; t < t_end; ++t) {
      const int c = (t * NW) >> 6;
      if (c != chunk) load(c);
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < NW; ++i) any |= w[i] = at(t * NW + i);
      if (any != 0) break;
    }
    return t;
  }
};

// One thread's share of a [rows][DH] tile on its way from memory to LDS: chunk id = tid + u threads.
template <typename T, int DH, int ROWS, int THREADS> struct Stage {
  typedef Geo<T, DH> Gm;
  static constexpr int N = ROWS * Gm::CPR / THREADS;
  static_assert(ROWS * Gm::CPR % THREADS == 0, "a thread stages whole chunks");
  u32x4 r[N];
  // Rows past `rows` load the last one, chunks past D the first: in range, and zeroed by put().
  __device__ __forceinline__ void get(const T* base, int64_t stride, int row0, int rows, int D) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int id = threadIdx.x + u * THREADS, row = id / Gm::CPR, ch = id % Gm::CPR;
      const int64_t off = (int64_t)min(row0 + row, rows - 1) * stride + (ch * Gm::EPC < D ? ch * Gm::EPC : 0);
      r[u] = *(const u32x4*)(base + off);
    }
  }
  // Rows whose bit in `w` is clear, and chunks past D, as zeros.
  template <int NW> __device__ __forceinline__ void put(char* tile, const uint32_t (&w)[NW], int D) const {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int id = threadIdx.x + u * THREADS, row = id / Gm::CPR, ch = id % Gm::CPR;
      uint32_t bits = w[0];
#pragma unroll
      for (int i = 1; i < NW; ++i) bits = (row >> 5) == i ? w[i] : bits;
      const bool on = ((bits >> (row & 31)) & 1) && ch * Gm::EPC < D;
      *(u32x4*)(tile + lds_at<T, DH>(row, ch)) = on ? r[u] : u32x4{0, 0, 0, 0};
    }
  }
};

// A row's fragments straight from memory (the operand that a wave keeps): chunk 2 c + half of each step.
template <typename T, int DH>
__device__ __forceinline__ void load_row(frag_t<T>* f, const T* row, int half, int D, bool on) {
  typedef Geo<T, DH> Gm;
#pragma unroll
  for (int c = 0; c < Gm::NC; ++c) {
    const int d = c * Gm::KC + half * Gm::EPC;
    const u32x4 v = *(const u32x4*)(row + (d < D ? d : 0));
    f[c] = __builtin_bit_cast(frag_t<T>, on && d < D ? v : u32x4{0, 0, 0, 0});
  }
}

// Four consecutive values of an output row.
template <typename T> struct Vec4;
template <> struct Vec4<bf16> { typedef bf16x4 type; };
template <> struct Vec4<f16> { typedef f16x4 type; };
template <> struct Vec4<float> { typedef f32x4 type; };
template <typename T> __device__ __forceinline__ void store4(T* p, const f32x16& a, int r, float f) {
  typename Vec4<T>::type o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = from_f32<T>(a[r + e] * f);
  *(typename Vec4<T>::type*)p = o;
}
// A transposed result column (the lane's row) to memory.
template <typename T, int DB>
__device__ __forceinline__ void store_col(T* row, const f32x16 (&acc)[DB], float f, int half, int D) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = db * 32 + reg_row(r) + 4 * half;
      if (d < D) store4<T>(row + d, acc[db], r, f);
    }
}

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.0f;
  return z;
}

// A lane's row of the packed rows [0, R): query head g of the group, position i.
struct Row {
  int g, i;
  bool in;
};
__device__ __forceinline__ Row row_of(const Params& p, int r) {
  Row w;
  w.in = r < p.R;
  const int rr = min(r, p.R - 1);
  w.g = p.G == 1 ? 0 : rr / p.Sq;
  w.i = rr - w.g * p.Sq;
  return w;
}
// Smallest and largest position among packed rows [r0, r1).
__device__ __forceinline__ void pos_range(const Params& p, int r0, int r1, int* lo, int* hi) {
  const int a = r0 / p.Sq, z = (min(r1, p.R) - 1) / p.Sq;
  *lo = a == z ? r0 - a * p.Sq : 0;
  *hi = a == z ? min(r1, p.R) - 1 - a * p.Sq : p.Sq - 1;
}

// ---- forward -----------------------------------------------------------------------------
// WR x WK waves: wave (wr, wk) holds 32 NB rows and takes the 32 JB keys wk of each tile of 32 JB WK.
// Each wave keeps its rows' running maximum and sum; where WK > 1 the waves' results are joined
// through LDS at the end, and with SPLIT each workgroup takes tiles_per_split tiles of the keys and
// writes its normalised result and log sum for attn_join_kernel.
template <typename T, int DH, int NB, int WR, int WK, int JB, int NBUF, bool SPLIT>
__global__ __launch_bounds__(64 * WR * WK, NB * DH > 128 ? 1 : 2) void attn_fwd_kernel(Params p) {
  typedef Geo<T, DH> Gm;
  constexpr int THREADS = 64 * WR * WK, BK = 32 * JB * WK, NW = JB * WK;
  constexpr int TILE = BK * Gm::ROW;
  static_assert(WK == 1 || (NB == 1 && WR == 1 && NBUF * 2 * TILE >= WK * 32 * DH * 4), "joining waves reuse the tiles");
  __shared__ __attribute__((aligned(16))) char smem[NBUF * 2 * TILE];
  __shared__ float wave_stat[WK > 1 ? 2 * WK * 32 : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int wr = wave % WR, wk = wave / WR;
  const int row_tiles = (p.R + 32 * NB * WR - 1) / (32 * NB * WR);
  int id = xcd_range(blockIdx.x, gridDim.x);
  const int split = SPLIT ? id % p.splits : 0;
  if (SPLIT) id /= p.splits;
  const int bh = id / row_tiles, tile = row_tiles - 1 - id % row_tiles;  // causal: longest first
  const int b = bh / p.Hk, hk = bh % p.Hk;
  const int r0 = tile * 32 * NB * WR;

  int i_lo, i_hi;
  pos_range(p, r0, r0 + 32 * NB * WR, &i_lo, &i_hi);
  const int off = p.Sk - p.Sq;
  const int kend = p.causal ? max(0, min(p.Sk, i_hi + off + 1)) : p.Sk;
  int t_end = (kend + BK - 1) / BK, t = -1;
  if (SPLIT) {
    t = split * p.tiles_per_split - 1;
    t_end = min(t_end, t + 1 + p.tiles_per_split);
  }

  Row row[NB];
  frag_t<T> qf[NB][Gm::NC];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    row[n] = row_of(p, r0 + (wr * NB + n) * 32 + (lane & 31));
    load_row<T, DH>(qf[n], (const T*)p.q + b * p.sq.b + (int64_t)(hk * p.G + row[n].g) * p.sq.h + row[n].i * p.sq.s,
                    half, p.D, true);
  }
  const T* kb = (const T*)p.k + b * p.sk.b + hk * p.sk.h;
  const T* vb = (const T*)p.v + b * p.sv.b + hk * p.sv.h;

  f32x16 acc[NB][Gm::DB];
  float m[NB], l[NB];  // the running maximum (times c) and this half's part of the sum
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.0f;
#pragma unroll
    for (int db = 0; db < Gm::DB; ++db) acc[n][db] = zero16();
  }

  KeyBits bits;
  bits.init(p, b, kend);
  uint32_t w[NW], wn[NW];
  t = bits.next<NW>(t, t_end, w);
  Stage<T, DH, BK, THREADS> ks, vs;
  if (t < t_end) {
    ks.get(kb, p.sk.s, t * BK, p.Sk, p.D);
    vs.get(vb, p.sv.s, t * BK, p.Sk, p.D);
    ks.template put<NW>(smem, w, p.D);
    vs.template put<NW>(smem + TILE, w, p.D);
    __syncthreads();
  }
  int buf = 0;
  while (t < t_end) {
    const int tn = bits.next<NW>(t, t_end, wn);
    if (tn < t_end) {
      ks.get(kb, p.sk.s, tn * BK, p.Sk, p.D);
      vs.get(vb, p.sv.s, tn * BK, p.Sk, p.D);
    }
    const char* kt = smem + buf * 2 * TILE;
    const char* vt = kt + TILE;
    f32x16 s[NB][JB];
#pragma unroll
    for (int jb = 0; jb < JB; ++jb) {
#pragma unroll
      for (int n = 0; n < NB; ++n) s[n][jb] = zero16();
#pragma unroll
      for (int c = 0; c < Gm::NC; ++c) {
        const frag_t<T> kf = lds_frag<T>(kt + lds_at<T, DH>((wk * JB + jb) * 32 + (lane & 31), 2 * c + half));
#pragma unroll
        for (int n = 0; n < NB; ++n) s[n][jb] = mma(kf, qf[n][c], s[n][jb]);
      }
    }
    uint32_t wj[JB];
    bool part = false;
#pragma unroll
    for (int jb = 0; jb < JB; ++jb) {
      wj[jb] = w[jb];
#pragma unroll
      for (int x = 1; x < WK; ++x) wj[jb] = wk == x ? w[x * JB + jb] : wj[jb];
      part |= wj[jb] != 0xffffffffu;
    }
    if (part) {
#pragma unroll
      for (int jb = 0; jb < JB; ++jb) {
        const uint32_t mine = wj[jb] >> (4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
          for (int n = 0; n < NB; ++n) s[n][jb][r] = (mine >> reg_row(r)) & 1 ? s[n][jb][r] : -INFINITY;
      }
    }
    if (p.causal && (t + 1) * BK - 1 > i_lo + off) {
#pragma unroll
      for (int jb = 0; jb < JB; ++jb)
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const int lim = row[n].i + off - (t * BK + (wk * JB + jb) * 32 + 4 * half);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[n][jb][r] = reg_row(r) <= lim ? s[n][jb][r] : -INFINITY;
        }
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float top = s[n][0][0];
#pragma unroll
      for (int jb = 0; jb < JB; ++jb)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[n][jb][r]);
      top = other_half_max(top) * p.c;
      // The maximum follows only where it has grown by more than 2^8 (p stays below 2^8, and sums
      // have room for that): after the first tiles the output's rescaling is hardly ever taken.
      const bool up = top > m[n] + 8.0f;
      if (__any(up)) {
        const float mn = up ? top : m[n];
        const float a = up ? __builtin_amdgcn_exp2f(m[n] - mn) : 1.0f;
        l[n] *= a;
#pragma unroll
        for (int db = 0; db < Gm::DB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[n][db][r] *= a;
        m[n] = mn;
      }
      const float mm = m[n] == -INFINITY ? 0.0f : m[n];
      float sum = 0.0f;
#pragma unroll
      for (int jb = 0; jb < JB; ++jb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[n][jb][r] = __builtin_amdgcn_exp2f(fmaf(s[n][jb][r], p.c, -mm));
          sum += s[n][jb][r];
        }
      l[n] += sum;
    }
#pragma unroll
    for (int jb = 0; jb < JB; ++jb)
#pragma unroll
      for (int c = 0; c < Gm::PB; ++c) {
        frag_t<T> pf[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) pf[n] = pack<T>(s[n][jb], c);
#pragma unroll
        for (int db = 0; db < Gm::DB; ++db) {
          const frag_t<T> vf = lds_cols<T, DH>(vt, (wk * JB + jb) * 32 + c * Gm::KC, db, lane);
#pragma unroll
          for (int n = 0; n < NB; ++n) acc[n][db] = mma(vf, pf[n], acc[n][db]);
        }
      }
    if (NBUF == 1) __syncthreads();
    if (tn < t_end) {
      if (NBUF == 2) buf ^= 1;
      ks.template put<NW>(smem + buf * 2 * TILE, wn, p.D);
      vs.template put<NW>(smem + buf * 2 * TILE + TILE, wn, p.D);
    }
    __syncthreads();
    t = tn;
#pragma unroll
    for (int i = 0; i < NW; ++i) w[i] = wn[i];
  }

#pragma unroll
  for (int n = 0; n < NB; ++n) l[n] = other_half_sum(l[n]);

  if constexpr (WK > 1) {
    // acc, m and l of the WK waves, each for the same 32 rows, to LDS; wave 0 joins them.
    __syncthreads();
    float* mine = (float*)smem + wave * 32 * DH;
#pragma unroll
    for (int db = 0; db < Gm::DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) mine[(db * 16 + r) * 64 + lane] = acc[0][db][r];
    if (half == 0) {
      wave_stat[wave * 64 + lane] = m[0];
      wave_stat[wave * 64 + 32 + lane] = l[0];
    }
    __syncthreads();
    if (wave > 0) return;
    float top = m[0];
#pragma unroll
    for (int x = 1; x < WK; ++x) top = fmaxf(top, wave_stat[x * 64 + (lane & 31)]);
    const float mm = top == -INFINITY ? 0.0f : top;
    float wt[WK], sum = 0.0f;
#pragma unroll
    for (int x = 0; x < WK; ++x) {
      wt[x] = __builtin_amdgcn_exp2f(wave_stat[x * 64 + (lane & 31)] - mm);
      sum += wt[x] * wave_stat[x * 64 + 32 + (lane & 31)];
    }
#pragma unroll
    for (int db = 0; db < Gm::DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float a = 0.0f;
#pragma unroll
        for (int x = 0; x < WK; ++x) a += wt[x] * ((const float*)smem)[x * 32 * DH + (db * 16 + r) * 64 + lane];
        acc[0][db][r] = a;
      }
    m[0] = top;
    l[0] = sum;
  }
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    if (!row[n].in) continue;
    const bool none = l[n] == 0.0f;
    const float inv = none ? 0.0f : 1.0f / l[n];
    const float lse = none ? -INFINITY : m[n] + __builtin_amdgcn_logf(l[n]);
    if constexpr (SPLIT) {
      const int64_t at = ((int64_t)bh * p.splits + split) * p.R + r0 + (wr * NB + n) * 32 + (lane & 31);
      store_col<float, Gm::DB>(p.part + at * p.D, acc[n], inv, half, p.D);
      if (half == 0) p.part_lse[at] = lse;
    } else {
      const int64_t h = hk * p.G + row[n].g;
      store_col<T, Gm::DB>((T*)p.out + b * p.so.b + h * p.so.h + row[n].i * p.so.s, acc[n], inv, half, p.D);
      if (half == 0 && p.lse != nullptr) p.lse[((int64_t)b * p.Hq + h) * p.Sq + row[n].i] = lse;
    }
  }
}

// The splits of a row joined: weights exp2(lse_s - max), one lane per split, then two columns per lane.
template <typename T>
__global__ __launch_bounds__(kThreads) void attn_join_kernel(Params p) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)p.B * p.Hk * p.R;
  const int64_t id = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (id >= n) return;
  const int r = (int)(id % p.R);
  const int64_t bh = id / p.R;
  const int64_t b = bh / p.Hk, hk = bh % p.Hk;
  const Row row = row_of(p, r);
  const float lse = lane < p.splits ? p.part_lse[(bh * p.splits + lane) * p.R + r] : -INFINITY;
  const float top = wave_max(lse), mm = top == -INFINITY ? 0.0f : top;
  const float wt = __builtin_amdgcn_exp2f(lse - mm);
  const float sum = wave_sum(wt);
  const int d = lane * 2;
  float a0 = 0.0f, a1 = 0.0f;
  const float* src = p.part + (bh * p.splits * p.R + r) * p.D + (d < p.D ? d : 0);
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float f = lane_f(wt, s);
    const float2 v = *(const float2*)(src + (int64_t)s * p.R * p.D);
    a0 += f * v.x;
    a1 += f * v.y;
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const int64_t h = hk * p.G + row.g;
  if (d < p.D) {
    T* o = (T*)p.out + b * p.so.b + h * p.so.h + row.i * p.so.s + d;
    o[0] = from_f32<T>(a0 * inv);
    o[1] = from_f32<T>(a1 * inv);
  }
  if (lane == 0 && p.lse != nullptr)
    p.lse[(b * p.Hq + h) * p.Sq + row.i] = sum == 0.0f ? -INFINITY : top + __builtin_amdgcn_logf(sum);
}

// ---- backward ----------------------------------------------------------------------------
// ds holds products of a probability and a gradient, which may lie below fp16's normal range (2^-14).
// In fp16 each column of ds (one row's in the dq kernel, one key's in the dk kernel) is therefore
// multiplied by a power of two that puts its largest value so far near 2^10; when a tile passes 2^14
// the column's sums are rescaled. Other types need no such factor.
template <typename T> struct ColScale {
  __device__ __forceinline__ float inv() const { return 1.0f; }
  template <int DB> __device__ __forceinline__ void apply(f32x16&, f32x16 (&)[DB]) {}
};
template <> struct ColScale<f16> {
  float f = 0x1p126f;
  __device__ __forceinline__ float inv() const { return 1.0f / f; }
  template <int DB> __device__ __forceinline__ void apply(f32x16& ds, f32x16 (&acc)[DB]) {
    float top = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(ds[r]));
    top = other_half_max(top);
    const bool up = top * f > 0x1p14f;
    if (__any(up)) {
      const int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
      const float fn = up ? __builtin_bit_cast(float, (uint32_t)(137 - max(e, -116)) << 23) : f;
      const float g = fn / f;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[db][r] *= g;
      f = fn;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) ds[r] *= f;
  }
};
// In fp16 the probabilities of the dv product carry a factor 2^10 for the same reason.
template <typename T> constexpr float kLog2Up = 0.0f;
template <> constexpr float kLog2Up<f16> = 10.0f;

// dq, and delta for the next kernel. Four waves of 32 NB rows each; the tiles as in the forward.
template <typename T, int DH, int NB, int JB, int NBUF>
__global__ __launch_bounds__(kThreads, 1) void attn_dq_kernel(Params p) {
  typedef Geo<T, DH> Gm;
  constexpr int BK = 32 * JB, TILE = BK * Gm::ROW;
  __shared__ __attribute__((aligned(16))) char smem[NBUF * 2 * TILE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int row_tiles = (p.R + 128 * NB - 1) / (128 * NB);
  const int id = xcd_range(blockIdx.x, gridDim.x);
  const int bh = id / row_tiles, tile = row_tiles - 1 - id % row_tiles;
  const int b = bh / p.Hk, hk = bh % p.Hk;
  const int r0 = tile * 128 * NB;
  int i_lo, i_hi;
  pos_range(p, r0, r0 + 128 * NB, &i_lo, &i_hi);
  const int off = p.Sk - p.Sq;
  const int kend = p.causal ? max(0, min(p.Sk, i_hi + off + 1)) : p.Sk;
  const int t_end = (kend + BK - 1) / BK;

  Row row[NB];
  frag_t<T> qf[NB][Gm::NC], gf[NB][Gm::NC];
  float lse[NB], delta[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    row[n] = row_of(p, r0 + (wave * NB + n) * 32 + (lane & 31));
    const int64_t h = hk * p.G + row[n].g;
    load_row<T, DH>(qf[n], (const T*)p.q + b * p.sq.b + h * p.sq.h + row[n].i * p.sq.s, half, p.D, true);
    load_row<T, DH>(gf[n], (const T*)p.dout + b * p.sdo.b + h * p.sdo.h + row[n].i * p.sdo.s, half, p.D, true);
    frag_t<T> of[Gm::NC];
    load_row<T, DH>(of, (const T*)p.o + b * p.so.b + h * p.so.h + row[n].i * p.so.s, half, p.D, true);
    float a = 0.0f;
#pragma unroll
    for (int c = 0; c < Gm::NC; ++c)
#pragma unroll
      for (int e = 0; e < Gm::EPC; ++e) a += to_f32(gf[n][c][e]) * to_f32(of[c][e]);
    delta[n] = other_half_sum(a);
    const int64_t at = ((int64_t)b * p.Hq + h) * p.Sq + row[n].i;
    lse[n] = p.lse[at];
    if (!row[n].in || lse[n] == -INFINITY) lse[n] = INFINITY;  // exp2(s - lse) = 0
    if (half == 0 && row[n].in) p.delta[at] = delta[n];
  }
  const T* kb = (const T*)p.k + b * p.sk.b + hk * p.sk.h;
  const T* vb = (const T*)p.v + b * p.sv.b + hk * p.sv.h;
  f32x16 acc[NB][Gm::DB];
  ColScale<T> cs[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int db = 0; db < Gm::DB; ++db) acc[n][db] = zero16();

  KeyBits bits;
  bits.init(p, b, kend);
  uint32_t w[JB], wn[JB];
  int t = bits.next<JB>(-1, t_end, w);
  Stage<T, DH, BK, kThreads> ks, vs;
  if (t < t_end) {
    ks.get(kb, p.sk.s, t * BK, p.Sk, p.D);
    vs.get(vb, p.sv.s, t * BK, p.Sk, p.D);
    ks.template put<JB>(smem, w, p.D);
    vs.template put<JB>(smem + TILE, w, p.D);
    __syncthreads();
  }
  int buf = 0;
  while (t < t_end) {
    const int tn = bits.next<JB>(t, t_end, wn);
    if (tn < t_end) {
      ks.get(kb, p.sk.s, tn * BK, p.Sk, p.D);
      vs.get(vb, p.sv.s, tn * BK, p.Sk, p.D);
    }
    const char* kt = smem + buf * 2 * TILE;
    const char* vt = kt + TILE;
#pragma unroll
    for (int jb = 0; jb < JB; ++jb) {
      f32x16 s[NB], dp[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) s[n] = dp[n] = zero16();
#pragma unroll
      for (int c = 0; c < Gm::NC; ++c) {
        const int at = lds_at<T, DH>(jb * 32 + (lane & 31), 2 * c + half);
        const frag_t<T> kf = lds_frag<T>(kt + at), vf = lds_frag<T>(vt + at);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          s[n] = mma(kf, qf[n][c], s[n]);
          dp[n] = mma(vf, gf[n][c], dp[n]);
        }
      }
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[n][r] = __builtin_amdgcn_exp2f(fmaf(s[n][r], p.c, -lse[n]));
      if (w[jb] != 0xffffffffu) {
        const uint32_t mine = w[jb] >> (4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
          for (int n = 0; n < NB; ++n) s[n][r] = (mine >> reg_row(r)) & 1 ? s[n][r] : 0.0f;
      }
      if (p.causal && t * BK + jb * 32 + 31 > i_lo + off) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const int lim = row[n].i + off - (t * BK + jb * 32 + 4 * half);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[n][r] = reg_row(r) <= lim ? s[n][r] : 0.0f;
        }
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[n][r] *= dp[n][r] - delta[n];
        cs[n].template apply<Gm::DB>(s[n], acc[n]);
      }
#pragma unroll
      for (int c = 0; c < Gm::PB; ++c) {
        frag_t<T> df[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) df[n] = pack<T>(s[n], c);
#pragma unroll
        for (int db = 0; db < Gm::DB; ++db) {
          const frag_t<T> kf = lds_cols<T, DH>(kt, jb * 32 + c * Gm::KC, db, lane);
#pragma unroll
          for (int n = 0; n < NB; ++n) acc[n][db] = mma(kf, df[n], acc[n][db]);
        }
      }
    }
    if (NBUF == 1) __syncthreads();
    if (tn < t_end) {
      if (NBUF == 2) buf ^= 1;
      ks.template put<JB>(smem + buf * 2 * TILE, wn, p.D);
      vs.template put<JB>(smem + buf * 2 * TILE + TILE, wn, p.D);
    }
    __syncthreads();
    t = tn;
#pragma unroll
    for (int i = 0; i < JB; ++i) w[i] = wn[i];
  }
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    if (!row[n].in) continue;
    const int64_t h = hk * p.G + row[n].g;
    store_col<T, Gm::DB>((T*)p.dq + b * p.sdq.b + h * p.sdq.h + row[n].i * p.sdq.s, acc[n], p.scale * cs[n].inv(), half,
                         p.D);
  }
}

// dk and dv. Four waves hold 32 NB keys each (K and V as right operands, in registers) and walk the
// rows of every query head of the group in tiles of 32 IB. A key that takes no part has its own
// column throughout, which is written as zeros: no element needs the key mask here.
template <typename T, int DH, int NB, int IB, int NBUF>
__global__ __launch_bounds__(kThreads, 1) void attn_dkv_kernel(Params p) {
  typedef Geo<T, DH> Gm;
  constexpr int BR = 32 * IB, TILE = BR * Gm::ROW;
  __shared__ __attribute__((aligned(16))) char smem[NBUF * 2 * TILE];
  __shared__ __attribute__((aligned(16))) float stat[NBUF * 2 * BR];  // lse, delta of the tile's rows
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int key_tiles = (p.Sk + 128 * NB - 1) / (128 * NB);
  const int id = xcd_range(blockIdx.x, gridDim.x);
  const int bh = id / key_tiles;
  const int b = bh / p.Hk, hk = bh % p.Hk;
  const int j0 = (id % key_tiles) * 128 * NB;
  const int off = p.Sk - p.Sq;

  // This workgroup's keys: which take part, and whether any does.
  int key[NB];
  bool on[NB];
  bool any = false;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    key[n] = j0 + (wave * NB + n) * 32 + (lane & 31);
    on[n] = key[n] < p.Sk;
    if (p.mask != nullptr) on[n] = key_on(p.mask, p.mask_dtype, b * p.mask_b + min(key[n], p.Sk - 1)) && on[n];
    any |= on[n];
  }
  const bool wave_any = __any(any);
  const bool wg_any = __syncthreads_or(any);

  f32x16 dk[NB][Gm::DB], dv[NB][Gm::DB];
  ColScale<T> cs[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int db = 0; db < Gm::DB; ++db) dk[n][db] = dv[n][db] = zero16();

  // Row tiles (g, it) of the group's heads; with `causal` those whose last row sees key j0.
  const int ntile = (p.Sq + BR - 1) / BR;
  const int first = p.causal ? min(ntile, max(0, j0 - off) / BR) : 0;
  if (wg_any && first < ntile) {
    frag_t<T> kf[NB][Gm::NC], vf[NB][Gm::NC];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int64_t j = min(key[n], p.Sk - 1);
      load_row<T, DH>(kf[n], (const T*)p.k + b * p.sk.b + hk * p.sk.h + j * p.sk.s, half, p.D, on[n]);
      load_row<T, DH>(vf[n], (const T*)p.v + b * p.sv.b + hk * p.sv.h + j * p.sv.s, half, p.D, on[n]);
    }
    Stage<T, DH, BR, kThreads> qs, gs;
    float st = 0.0f;  // threads [0, BR): lse, [BR, 2 BR): delta of the staged rows
    const auto get = [&](int g, int it) {
      const int64_t h = hk * p.G + g;
      qs.get((const T*)p.q + b * p.sq.b + h * p.sq.h, p.sq.s, it * BR, p.Sq, p.D);
      gs.get((const T*)p.dout + b * p.sdo.b + h * p.sdo.h, p.sdo.s, it * BR, p.Sq, p.D);
      if (threadIdx.x < 2 * BR) {
        const int i = it * BR + (threadIdx.x & (BR - 1));
        const float* src = threadIdx.x < BR ? p.lse : p.delta;
        st = src[((int64_t)b * p.Hq + h) * p.Sq + min(i, p.Sq - 1)];
        if (threadIdx.x < BR) st = i >= p.Sq || st == -INFINITY ? INFINITY : st - kLog2Up<T>;
        else st = i >= p.Sq ? 0.0f : st;
      }
    };
    const auto put = [&](int buf, int it) {
      uint32_t w[IB];
#pragma unroll
      for (int i = 0; i < IB; ++i) {
        const int left = p.Sq - it * BR - i * 32;
        w[i] = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
      }
      qs.template put<IB>(smem + buf * 2 * TILE, w, p.D);
      gs.template put<IB>(smem + buf * 2 * TILE + TILE, w, p.D);
      if (threadIdx.x < 2 * BR) stat[buf * 2 * BR + threadIdx.x] = st;
    };
    int g = 0, it = first, buf = 0;
    get(g, it);
    put(0, it);
    __syncthreads();
    while (g < p.G) {
      int gn = g, itn = it + 1;
      if (itn == ntile) {
        itn = first;
        ++gn;
      }
      if (gn < p.G) get(gn, itn);
      if (wave_any) {
        const char* qt = smem + buf * 2 * TILE;
        const char* gt = qt + TILE;
#pragma unroll
        for (int ib = 0; ib < IB; ++ib) {
          f32x16 s[NB], dp[NB];
#pragma unroll
          for (int n = 0; n < NB; ++n) s[n] = dp[n] = zero16();
#pragma unroll
          for (int c = 0; c < Gm::NC; ++c) {
            const int at = lds_at<T, DH>(ib * 32 + (lane & 31), 2 * c + half);
            const frag_t<T> qf = lds_frag<T>(qt + at), gf = lds_frag<T>(gt + at);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
              s[n] = mma(qf, kf[n][c], s[n]);
              dp[n] = mma(gf, vf[n][c], dp[n]);
            }
          }
          const float* lse = stat + buf * 2 * BR + ib * 32 + 4 * half;
          const float* del = lse + BR;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 l4 = *(const f32x4*)(lse + 8 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int n = 0; n < NB; ++n)
                s[n][4 * q + e] = __builtin_amdgcn_exp2f(fmaf(s[n][4 * q + e], p.c, -l4[e]));
          }
          const int i0 = it * BR + ib * 32 + 4 * half;
          if (p.causal && it * BR + ib * 32 < j0 + 128 * NB - 1 - off) {
#pragma unroll
            for (int n = 0; n < NB; ++n) {
              const int lim = key[n] - off - i0;  // rows from here on see the key
#pragma unroll
              for (int r = 0; r < 16; ++r) s[n][r] = reg_row(r) >= lim ? s[n][r] : 0.0f;
            }
          }
#pragma unroll
          for (int c = 0; c < Gm::PB; ++c) {
            frag_t<T> pf[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) pf[n] = pack<T>(s[n], c);
#pragma unroll
            for (int db = 0; db < Gm::DB; ++db) {
              const frag_t<T> gf = lds_cols<T, DH>(gt, ib * 32 + c * Gm::KC, db, lane);
#pragma unroll
              for (int n = 0; n < NB; ++n) dv[n][db] = mma(gf, pf[n], dv[n][db]);
            }
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 d4 = *(const f32x4*)(del + 8 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int n = 0; n < NB; ++n) s[n][4 * q + e] *= dp[n][4 * q + e] - d4[e];
          }
#pragma unroll
          for (int n = 0; n < NB; ++n) cs[n].template apply<Gm::DB>(s[n], dk[n]);
#pragma unroll
          for (int c = 0; c < Gm::PB; ++c) {
            frag_t<T> df[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) df[n] = pack<T>(s[n], c);
#pragma unroll
            for (int db = 0; db < Gm::DB; ++db) {
              const frag_t<T> qf = lds_cols<T, DH>(qt, ib * 32 + c * Gm::KC, db, lane);
#pragma unroll
              for (int n = 0; n < NB; ++n) dk[n][db] = mma(qf, df[n], dk[n][db]);
            }
          }
        }
      }
      if (NBUF == 1) __syncthreads();
      if (gn < p.G) {
        if (NBUF == 2) buf ^= 1;
        put(buf, itn);
      }
      __syncthreads();
      g = gn;
      it = itn;
    }
  }
  const float up = __builtin_amdgcn_exp2f(-kLog2Up<T>);
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    if (key[n] >= p.Sk) continue;
    if (!on[n]) {
#pragma unroll
      for (int db = 0; db < Gm::DB; ++db) dk[n][db] = dv[n][db] = zero16();
    }
    store_col<T, Gm::DB>((T*)p.dk + b * p.sdk.b + hk * p.sdk.h + key[n] * p.sdk.s, dk[n], p.scale * up * cs[n].inv(), half,
                         p.D);
    store_col<T, Gm::DB>((T*)p.dv + b * p.sdv.b + hk * p.sdv.h + key[n] * p.sdv.s, dv[n], up, half, p.D);
  }
}

// ---- launches ----------------------------------------------------------------------------
constexpr int64_t kTargetGroups = 512;  // workgroups that fill the chip twice

struct FwdPlan {
  bool few;  // at most 32 rows look at a key head: waves share the keys
  int nb, splits, tiles_per_split;
  int64_t groups;
};

// Keys are split where there are few workgroups and each has many tiles.
FwdPlan fwd_plan(int64_t B, int64_t Hk, int64_t R, int64_t Sk, int64_t D, int es) {
  FwdPlan f;
  f.few = R <= 32;
  f.nb = !f.few && es == 2 && D <= 64 && B * Hk * cdiv(R, 256) >= kTargetGroups ? 2 : 1;
  const int64_t rows = f.few ? 32 : 128 * f.nb;
  f.groups = B * Hk * cdiv(R, rows);
  const int64_t tiles = cdiv(Sk, f.few ? 128 : 64);
  int64_t n = std::min<int64_t>({cdiv(kTargetGroups, std::max<int64_t>(f.groups, 1)), std::max<int64_t>(tiles / 4, 1), kMaxSplits});
  f.tiles_per_split = (int)cdiv(tiles, n);
  f.splits = (int)cdiv(tiles, f.tiles_per_split);
  return f;
}

size_t fwd_bytes(const FwdPlan& f, int64_t B, int64_t Hk, int64_t R, int64_t D) {
  return f.splits > 1 ? (size_t)(B * Hk * f.splits * R) * (size_t)(D + 1) * 4 : 0;
}

template <typename T, int DH>
void launch_fwd(const FwdPlan& f, const Params& p, hipStream_t st) {
  const dim3 grid((unsigned)(f.groups * f.splits)), block(kThreads);
  if (f.few) {
    if (f.splits > 1) hipLaunchKernelGGL((attn_fwd_kernel<T, DH, 1, 1, 4, 1, 1, true>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((attn_fwd_kernel<T, DH, 1, 1, 4, 1, 1, false>), grid, block, 0, st, p);
  } else if (f.nb == 1) {
    if (f.splits > 1) hipLaunchKernelGGL((attn_fwd_kernel<T, DH, 1, 4, 1, 2, 2, true>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((attn_fwd_kernel<T, DH, 1, 4, 1, 2, 2, false>), grid, block, 0, st, p);
  } else if constexpr (sizeof(T) == 2 && DH <= 64) {
    hipLaunchKernelGGL((attn_fwd_kernel<T, DH, 2, 4, 1, 2, 2, false>), grid, block, 0, st, p);
  }
  if (f.splits > 1)
    hipLaunchKernelGGL(attn_join_kernel<T>, dim3((unsigned)cdiv((int64_t)p.B * p.Hk * p.R, kThreads / 64)), block, 0, st, p);
}

template <typename T, int DH>
void launch_bwd(const Params& p, hipStream_t st) {
  const int64_t bh = (int64_t)p.B * p.Hk;
  const dim3 block(kThreads);
  if (p.R > 0)
    hipLaunchKernelGGL((attn_dq_kernel<T, DH, 1, 2, 2>), dim3((unsigned)(bh * cdiv(p.R, 128))), block, 0, st, p);
  if (p.Sk > 0)
    hipLaunchKernelGGL((attn_dkv_kernel<T, DH, 1, 2, 2>), dim3((unsigned)(bh * cdiv(p.Sk, 128))), block, 0, st, p);
}

template <typename T> void fwd_t(const FwdPlan& f, const Params& p, hipStream_t st) {
  if (p.D <= 32) launch_fwd<T, 32>(f, p, st);
  else if (p.D <= 64) launch_fwd<T, 64>(f, p, st);
  else launch_fwd<T, 128>(f, p, st);
}
template <typename T> void bwd_t(const Params& p, hipStream_t st) {
  if (p.D <= 32) launch_bwd<T, 32>(p, st);
  else if (p.D <= 64) launch_bwd<T, 64>(p, st);
  else launch_bwd<T, 128>(p, st);
}

Strides strides(const int64_t* s) { return Strides{s[0], s[1], s[2]}; }

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// A tensor [B, H, S, D] that is read and written in 16-byte pieces: its base and the strides of the
// dimensions that it has more than one of.
bool tensor_ok(const void* p, const int64_t* s, int64_t B, int64_t H, int64_t S, int es) {
  const int64_t unit = 16 / es;
  return aligned(p, 16) && (B == 1 || s[0] % unit == 0) && (H == 1 || s[1] % unit == 0) && (S == 1 || s[2] % unit == 0);
}

// Status of a description, and its parameters: SPARTON_OK with *empty set where there is nothing to do.
int read_desc(const sparton_attention_desc* d, const void* mask, Params* p, bool* empty) {
  *empty = false;
  if (d == nullptr) return SPARTON_EINVAL;
  if (d->B < 0 || d->Hq < 0 || d->Hk < 0 || d->Sq < 0 || d->Sk < 0 || d->D <= 0) return SPARTON_EINVAL;
  if (d->dtype < SPARTON_F32 || d->dtype > SPARTON_F16) return SPARTON_EINVAL;
  if (mask != nullptr && (d->mask_dtype < SPARTON_MASK_I64 || d->mask_dtype > SPARTON_MASK_U8)) return SPARTON_EINVAL;
  if (!(d->scale > 0.0f) || isinf(d->scale)) return SPARTON_EINVAL;
  const int es = d->dtype == SPARTON_F32 ? 4 : 2;
  if (d->D * es % 16 != 0) return SPARTON_EINVAL;
  if (d->D > 128) return SPARTON_EUNSUPPORTED;
  if (d->B == 0 || d->Hq == 0) {
    *empty = true;
    return SPARTON_OK;
  }
  if (d->Hk == 0 || d->Hq % d->Hk != 0) return SPARTON_EINVAL;
  const int64_t lim = INT32_MAX, G = d->Hq / d->Hk;
  // Positions, packed rows and workgroup numbers (at most 64 splits) are 32-bit.
  if (d->B > lim || d->Hq > lim || d->Sq > lim / 2 || d->Sk > lim / 2 || G > (lim / 2) / std::max<int64_t>(d->Sq, 1))
    return SPARTON_EUNSUPPORTED;
  if (d->B > lim / d->Hq || d->B * d->Hk > (lim / kMaxSplits) / std::max({cdiv(G * d->Sq, 32), cdiv(d->Sk, 128), (int64_t)1}))
    return SPARTON_EUNSUPPORTED;
  p->mask = mask;
  p->sq = strides(d->q);
  p->sk = strides(d->k);
  p->sv = strides(d->v);
  p->so = strides(d->o);
  p->sdo = strides(d->d_o);
  p->sdq = strides(d->d_q);
  p->sdk = strides(d->d_k);
  p->sdv = strides(d->d_v);
  p->mask_b = d->mask_batch;
  p->B = (int)d->B;
  p->Hq = (int)d->Hq;
  p->Hk = (int)d->Hk;
  p->G = (int)G;
  p->Sq = (int)d->Sq;
  p->Sk = (int)d->Sk;
  p->D = (int)d->D;
  p->R = (int)(G * d->Sq);
  p->mask_dtype = d->mask_dtype;
  p->causal = d->causal != 0;
  p->scale = d->scale;
  p->c = d->scale * kLog2e;
  p->splits = 1;
  return SPARTON_OK;
}

}  // namespace attn
}  // namespace sparton

using namespace sparton;

#define SPARTON_EXPORT extern "C" __attribute__((visibility("default")))

SPARTON_EXPORT size_t sparton_attention_workspace_bytes(const sparton_attention_desc* d) {
  attn::Params p;
  bool empty;
  if (attn::read_desc(d, nullptr, &p, &empty) != SPARTON_OK || empty || p.R == 0 || p.Sk == 0) return 0;
  const int es = d->dtype == SPARTON_F32 ? 4 : 2;
  return attn::fwd_bytes(attn::fwd_plan(p.B, p.Hk, p.R, p.Sk, p.D, es), p.B, p.Hk, p.R, p.D);
}

SPARTON_EXPORT int sparton_attention_fwd(const sparton_attention_desc* d, const void* q, const void* k, const void* v,
                                         const void* mask, void* out, float* lse, void* workspace,
                                         size_t workspace_bytes, void* stream) {
  attn::Params p = {};
  bool empty;
  const int rc = attn::read_desc(d, mask, &p, &empty);
  if (rc != SPARTON_OK || empty || p.R == 0) return rc;
  if (q == nullptr || out == nullptr || (p.Sk > 0 && (k == nullptr || v == nullptr))) return SPARTON_EINVAL;
  const int es = d->dtype == SPARTON_F32 ? 4 : 2;
  if (!attn::tensor_ok(q, d->q, d->B, d->Hq, d->Sq, es) || !attn::tensor_ok(out, d->o, d->B, d->Hq, d->Sq, es) ||
      !attn::tensor_ok(k, d->k, d->B, d->Hk, d->Sk, es) || !attn::tensor_ok(v, d->v, d->B, d->Hk, d->Sk, es))
    return SPARTON_EALIGN;
  attn::FwdPlan f = attn::fwd_plan(p.B, p.Hk, p.R, std::max(p.Sk, 1), p.D, es);
  const size_t need = attn::fwd_bytes(f, p.B, p.Hk, p.R, p.D);
  if (need > 0) {
    if (workspace == nullptr || workspace_bytes < need) return SPARTON_EWORKSPACE;
    if (!attn::aligned(workspace, 256)) return SPARTON_EALIGN;
  }
  p.q = q;
  p.k = k;
  p.v = v;
  p.out = out;
  p.lse = lse;
  p.splits = f.splits;
  p.tiles_per_split = f.tiles_per_split;
  p.part = (float*)workspace;
  p.part_lse = p.part + (int64_t)p.B * p.Hk * f.splits * p.R * p.D;
  hipStream_t st = (hipStream_t)stream;
  if (d->dtype == SPARTON_BF16) attn::fwd_t<bf16>(f, p, st);
  else if (d->dtype == SPARTON_F16) attn::fwd_t<f16>(f, p, st);
  else attn::fwd_t<float>(f, p, st);
  return (int)hipGetLastError();
}

SPARTON_EXPORT size_t sparton_attention_bwd_workspace_bytes(const sparton_attention_desc* d) {
  attn::Params p;
  bool empty;
  if (attn::read_desc(d, nullptr, &p, &empty) != SPARTON_OK || empty) return 0;
  return (size_t)p.B * p.Hq * p.Sq * 4;
}

SPARTON_EXPORT int sparton_attention_bwd(const sparton_attention_desc* d, const void* q, const void* k, const void* v,
                                         const void* mask, const void* out, const float* lse, const void* d_out,
                                         void* d_q, void* d_k, void* d_v, void* workspace, size_t workspace_bytes,
                                         void* stream) {
  attn::Params p = {};
  bool empty;
  const int rc = attn::read_desc(d, mask, &p, &empty);
  if (rc != SPARTON_OK || empty) return rc;
  if ((p.R > 0 && (q == nullptr || out == nullptr || lse == nullptr || d_out == nullptr || d_q == nullptr)) ||
      (p.Sk > 0 && (k == nullptr || v == nullptr || d_k == nullptr || d_v == nullptr)))
    return SPARTON_EINVAL;
  const int es = d->dtype == SPARTON_F32 ? 4 : 2;
  if (!attn::tensor_ok(q, d->q, d->B, d->Hq, d->Sq, es) || !attn::tensor_ok(out, d->o, d->B, d->Hq, d->Sq, es) ||
      !attn::tensor_ok(d_out, d->d_o, d->B, d->Hq, d->Sq, es) || !attn::tensor_ok(d_q, d->d_q, d->B, d->Hq, d->Sq, es) ||
      !attn::tensor_ok(k, d->k, d->B, d->Hk, d->Sk, es) || !attn::tensor_ok(v, d->v, d->B, d->Hk, d->Sk, es) ||
      !attn::tensor_ok(d_k, d->d_k, d->B, d->Hk, d->Sk, es) || !attn::tensor_ok(d_v, d->d_v, d->B, d->Hk, d->Sk, es))
    return SPARTON_EALIGN;
  const size_t need = (size_t)p.B * p.Hq * p.Sq * 4;
  if (need > 0) {
    if (workspace == nullptr || workspace_bytes < need) return SPARTON_EWORKSPACE;
    if (!attn::aligned(workspace, 256)) return SPARTON_EALIGN;
  }
  p.q = q;
  p.k = k;
  p.v = v;
  p.o = out;
  p.lse = const_cast<float*>(lse);
  p.delta = (float*)workspace;
  p.dout = d_out;
  p.dq = d_q;
  p.dk = d_k;
  p.dv = d_v;
  hipStream_t st = (hipStream_t)stream;
  if (d->dtype == SPARTON_BF16) attn::bwd_t<bf16>(p, st);
  else if (d->dtype == SPARTON_F16) attn::bwd_t<f16>(p, st);
  else attn::bwd_t<float>(p, st);
  return (int)hipGetLastError();
}
