// Attention of a backbone layer, forward and backward, on gfx950:
//     s_ij = scale q_i . k_j            over the keys j that row i may look at
//     p_ij = exp(s_ij - L_i),  L_i = log sum_j exp(s_ij),   o_i = sum_j p_ij v_j
//     delta_i = do_i . o_i,   ds_ij = p_ij (do_i . v_j - delta_i)
//     dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
// A key takes part where the key mask is nonzero and, with `causal`, where j <= i + Sk - Sq. Query
// head h reads key head h / (Hq / Hk); dk and dv are summed over the heads that share one. A row with
// no key gives o = 0 and zero gradients. A key that the mask drops is replaced by zeros: what its memory
// holds (NaN, infinities) reaches no output. A pair that `causal` hides while another row of the tile sees
// the key is multiplied, with p = 0: there 0 * NaN is NaN.
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
// A launch holds fewer than 2^32 threads (past that, workgroups were left out without an error).
constexpr int64_t kMaxGroups = (((int64_t)1 << 32) - 1) / kThreads;

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

// LDS rows are ROW bytes; the chunks of row r are permuted by XOR with f(r), which has period 16 at
// most. It serves both reads: one chunk of 8 consecutive rows (a row operand) and 64 bytes of 4
// consecutive rows (a column operand) each fall on different banks.
template <int ROW> __device__ __forceinline__ int swz(int r) {
  if constexpr (ROW == 64) return (r >> 1) & 3;
  else if constexpr (ROW == 128) return ((r & 2) << 1) | ((r & 4) >> 1) | (r & 1);
  else return ((r & 3) << 2) | ((r >> 2) & 3);
}
template <typename T, int DH> __device__ __forceinline__ int lds_at(int row, int chunk) {
  typedef Geo<T, DH> Gm;
  return row * Gm::ROW + ((chunk ^ swz<Gm::ROW>(row)) << 4);
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

// Probabilities and ds reach below fp16's normal range (2^-14), where they would lose bits, or all of them
// while the row's sum still counts them. In fp16 the forward's, which are at most 2^8 (see below), carry a
// factor 2^7, the dv product's, which are at most 1, 2^10, and ds one of its column (see ColScale).
template <typename T> constexpr float kLog2UpFwd = 0.0f;
template <> constexpr float kLog2UpFwd<f16> = 7.0f;
template <typename T> constexpr float kDownFwd = 1.0f;
template <> constexpr float kDownFwd<f16> = 0x1p-7f;
template <typename T> constexpr float kLog2Up = 0.0f;
template <> constexpr float kLog2Up<f16> = 10.0f;

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

// Workgroup w's place among `pairs` (batch row, key head) pairs of `tiles` workgroups each. Consecutive
// workgroups go to the eight XCDs in turn. A pair's tiles stay on one XCD, whose L2 then holds its keys
// and values, and the pairs go round the XCDs, so that long and short rows of a padded batch spread
// evenly; what is left of pairs after whole rounds is cut into eight runs of tiles. With `causal` tiles
// differ in length: an XCD then takes all its pairs' longest tiles first (by_tile), which leaves the
// short ones for the end, and what is shared is read from beyond the L2. 16 x 32 heads over 8 key heads,
// 512 x 512 x 128, padded: forward 95 -> 82 us, dq 120 -> 106, dk and dv 214 -> 148; 8 x 16 heads of
// 2048 x 2048 x 64: 142 -> 123, 174 -> 150, 223 -> 192. Tiles of one length lose by it: 8 x 12 heads of
// 512 x 512, dq 23.4 -> 25.5.
struct Place {
  int pair, tile;
};
__device__ __forceinline__ Place place_of(int w, int pairs, int tiles, bool by_tile) {
  const int x = w & 7, k = w >> 3, rounds = pairs >> 3, whole = rounds * tiles;
  Place p;
  if (k < whole) {
    p.pair = (by_tile ? k % rounds : k / tiles) * 8 + x;
    p.tile = by_tile ? k / rounds : k % tiles;
  } else {
    const int n = (pairs & 7) * tiles, i = x * (n >> 3) + min(x, n & 7) + (k - whole);
    p.pair = rounds * 8 + i / tiles;
    p.tile = i % tiles;
  }
  return p;
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
  // Eight loads are in flight at a time: one after the other would cost a round trip per 64 keys.
  template <typename M> __device__ __forceinline__ void gather(int k0, int n) {
    const int lane = threadIdx.x & 63;
    for (int x0 = 0; x0 < n; x0 += 8) {
      M v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = ((const M*)mask)[row + min(k0 + (x0 + i) * 64 + lane, kend - 1)];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int x = x0 + i;
        const uint64_t bits = __ballot(v[i] != 0 && k0 + x * 64 + lane < kend);
        word = lane == 2 * x ? (uint32_t)bits : lane == 2 * x + 1 ? (uint32_t)(bits >> 32) : word;
      }
    }
  }
  __device__ __forceinline__ void load(int c) {  // keys [2048 c, 2048 (c + 1)), below kend
    const int k0 = c * 2048, n = min(32, (kend - k0 + 63) >> 6);
    chunk = c;
    word = 0;
    if (mask == nullptr) {
      const int left = kend - k0 - (threadIdx.x & 63) * 32;
      word = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
    } else if (dtype == SPARTON_MASK_I64) gather<int64_t>(k0, n);
    else if (dtype == SPARTON_MASK_I32) gather<int32_t>(k0, n);
    else gather<uint8_t>(k0, n);
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
  // Whether no tile after t, below t_end, has a key (false where that takes another load of the mask).
  template <int NW> __device__ __forceinline__ bool last(int t, int t_end) const {
    return (t_end * NW - 1) >> 6 == chunk && !__any(word != 0 && (int)(threadIdx.x & 63) > ((t * NW + NW - 1) & 63));
  }
};

// What a staged chunk is read from past the last row and past D: every load is then unconditional.
__device__ u32x4 zero_chunk;

// One thread's share of a [ROWS][DH] tile on its way from memory to LDS: chunk `ch` of rows row0 + u RPU.
template <typename T, int DH, int ROWS, int THREADS> struct Stage {
  typedef Geo<T, DH> Gm;
  static constexpr int N = ROWS * Gm::CPR / THREADS;
  static constexpr int RPU = THREADS / Gm::CPR;
  static_assert(ROWS * Gm::CPR % THREADS == 0 && THREADS % Gm::CPR == 0, "a thread stages whole chunks of one column");
  u32x4 r[N];
  const T* mine;
  int64_t stride;
  int row0, ch, rows;  // rows: how many there are for this chunk (none past D)
  __device__ __forceinline__ void init(const T* base, int64_t stride_, int rows_, int D) {
    row0 = threadIdx.x / Gm::CPR;
    ch = threadIdx.x % Gm::CPR;
    rows = ch * Gm::EPC < D ? rows_ : 0;
    stride = stride_;
    mine = base + row0 * stride + ch * Gm::EPC;
  }
  __device__ __forceinline__ void get(int first) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const T* at = mine + (int64_t)(first + u * RPU) * stride;
      r[u] = *(first + row0 + u * RPU < rows ? (const u32x4*)at : &zero_chunk);
    }
  }
  __device__ __forceinline__ int to(int u) const {
    return RPU % 16 == 0 ? lds_at<T, DH>(row0, ch) + u * RPU * Gm::ROW : lds_at<T, DH>(row0 + u * RPU, ch);
  }
  __device__ __forceinline__ void put(char* tile) const {
#pragma unroll
    for (int u = 0; u < N; ++u) *(u32x4*)(tile + to(u)) = r[u];
  }
  // Rows whose bit in `w` is clear become zeros.
  template <int NW> __device__ __forceinline__ void clear(const uint32_t (&w)[NW]) {
    uint32_t all = w[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) all &= w[i];
    if (all == 0xffffffffu) return;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int row = row0 + u * RPU;
      uint32_t bits = w[0];
#pragma unroll
      for (int i = 1; i < NW; ++i) bits = (row >> 5) == i ? w[i] : bits;
      if (!((bits >> (row & 31)) & 1)) r[u] = u32x4{0, 0, 0, 0};
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
// WR x WK waves: wave (wr, wk) holds 32 rows and takes the 32 JB keys wk of each tile of 32 JB WK.
// Each wave keeps its rows' running maximum and sum; where WK > 1 the results of a row's waves are joined
// through LDS at the end, and with SPLIT each workgroup takes tiles_per_split tiles of the keys and
// writes its normalised result and log sum for attn_join_kernel.
//
// What bounds it. Long rows (12 heads of 8192 x 8192 x 64, bf16): 270 us, 760 TFLOP/s, half of what a
// large library product reaches on the card: 32 x 32 scores take eight MFMAs of 32 cycles, 16
// exponentials of 8, and some 60 maxima, multiply-adds, sums and conversions of 4 cycles or less. Three
// waves a SIMD (149 registers; 768 workgroups) overlap the matrix and the vector unit only in part: the
// matrix unit is busy 39% of the time, and so is the LDS, of which each fragment feeds one MFMA. Short rows (padded 32 x 12 heads
// of 256 x 256: 18 us) pay for the way to the first tile, four tiles being all there are. A
// token against a long cache (4 x 8 key heads of 20001 x 128, 9000 or more in use) is bound by memory:
// 50 us, 4.7 TB/s, though at head size 128 the four waves that share a row block spill 36 to 40 registers a
// lane in 16 bits, and in fp32 hold one wave a SIMD (all 20001 keys: 190 us, 3.4 TB/s). The tile's keys
// pass from memory through registers to two LDS buffers, so that the next tile's loads run under this one's
// products and a masked key's memory can be replaced by zeros.
template <typename T, int DH, int WR, int WK, int JB, int NBUF, bool SPLIT>
__global__ __launch_bounds__(64 * WR * WK, sizeof(T) * DH <= 256 ? 2 : 1) void attn_fwd_kernel(Params p) {
  typedef Geo<T, DH> Gm;
  constexpr int THREADS = 64 * WR * WK, BK = 32 * JB * WK, NW = JB * WK;
  constexpr int TILE = BK * Gm::ROW;
  static_assert(WK == 1 || NBUF * 2 * TILE >= WR * WK * 32 * DH * 4, "joining waves reuse the tiles");
  __shared__ __attribute__((aligned(16))) char smem[NBUF * 2 * TILE];
  __shared__ float wave_stat[WK > 1 ? WR * WK * 64 : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int wr = wave % WR, wk = wave / WR;
  const int row_tiles = (p.R + 32 * WR - 1) / (32 * WR);
  const Place at = place_of(blockIdx.x, p.B * p.Hk, SPLIT ? row_tiles * p.splits : row_tiles, p.causal);
  const int split = SPLIT ? at.tile % p.splits : 0;
  const int bh = at.pair, tile = row_tiles - 1 - (SPLIT ? at.tile / p.splits : at.tile);  // causal: longest first
  const int b = bh / p.Hk, hk = bh % p.Hk;
  const int r0 = tile * 32 * WR;

  int i_lo, i_hi;
  pos_range(p, r0, r0 + 32 * WR, &i_lo, &i_hi);
  const int off = p.Sk - p.Sq;
  const int kend = p.causal ? max(0, min(p.Sk, i_hi + off + 1)) : p.Sk;
  int t_end = (kend + BK - 1) / BK, t = -1;
  if (SPLIT) {
    t = split * p.tiles_per_split - 1;
    t_end = min(t_end, t + 1 + p.tiles_per_split);
  }

  const Row row = row_of(p, r0 + wr * 32 + (lane & 31));
  frag_t<T> qf[Gm::NC];
  load_row<T, DH>(qf, (const T*)p.q + b * p.sq.b + (int64_t)(hk * p.G + row.g) * p.sq.h + row.i * p.sq.s, half, p.D, true);
  const T* kb = (const T*)p.k + b * p.sk.b + hk * p.sk.h;
  const T* vb = (const T*)p.v + b * p.sv.b + hk * p.sv.h;

  f32x16 acc[Gm::DB];
  float m = -INFINITY, l = 0.0f;  // the running maximum (times c) and this half's part of the sum
#pragma unroll
  for (int db = 0; db < Gm::DB; ++db) acc[db] = zero16();

  // The first tile is on its way before the mask is known, which seldom leaves it out.
  Stage<T, DH, BK, THREADS> ks, vs;
  ks.init(kb, p.sk.s, p.Sk, p.D);
  vs.init(vb, p.sv.s, p.Sk, p.D);
  const int ahead = t + 1;
  ks.get(ahead * BK);
  vs.get(ahead * BK);
  KeyBits bits;
  bits.init(p, b, kend);
  uint32_t w[NW], wn[NW];
  t = bits.next<NW>(t, t_end, w);
  if (t < t_end) {
    if (t != ahead) {
      ks.get(t * BK);
      vs.get(t * BK);
    }
    ks.template clear<NW>(w);
    vs.template clear<NW>(w);
    ks.put(smem);
    vs.put(smem + TILE);
    __syncthreads();
  }
  int buf = 0;
  while (t < t_end) {
    const int tn = bits.next<NW>(t, t_end, wn);
    if (tn < t_end) {
      ks.get(tn * BK);
      vs.get(tn * BK);
    }
    const char* kt = smem + buf * 2 * TILE;
    const char* vt = kt + TILE;
    f32x16 s[JB];
#pragma unroll
    for (int jb = 0; jb < JB; ++jb) {
      s[jb] = zero16();
      frag_t<T> kf[Gm::NC];
#pragma unroll
      for (int c = 0; c < Gm::NC; ++c)
        kf[c] = lds_frag<T>(kt + lds_at<T, DH>((wk * JB + jb) * 32 + (lane & 31), 2 * c + half));
#pragma unroll
      for (int c = 0; c < Gm::NC; ++c) s[jb] = mma(kf[c], qf[c], s[jb]);
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
        for (int r = 0; r < 16; ++r) s[jb][r] = (mine >> reg_row(r)) & 1 ? s[jb][r] : -INFINITY;
      }
    }
    if (p.causal && (t + 1) * BK - 1 > i_lo + off) {
#pragma unroll
      for (int jb = 0; jb < JB; ++jb) {
        const int lim = row.i + off - (t * BK + (wk * JB + jb) * 32 + 4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[jb][r] = reg_row(r) <= lim ? s[jb][r] : -INFINITY;
      }
    }
    // From here to the tile's end a wave goes before the CU's others: they are then in their products
    // while this one is in its exponentials, where equal waves keep step and wait for the same unit
    // (8192 x 8192, 12 heads of 64: 291 -> 270 us).
    __builtin_amdgcn_s_setprio(1);
    float top = s[0][0];
#pragma unroll
    for (int jb = 0; jb < JB; ++jb)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[jb][r]);
    top = other_half_max(top) * p.c;
    // The maximum follows only where it has grown by more than 2^8 (p stays below 2^8, and sums
    // have room for that): after the first tiles the output's rescaling is hardly ever taken.
    const bool up = top > m + 8.0f;
    if (__any(up)) {
      const float mn = up ? top : m;
      const float a = up ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
      l *= a;
#pragma unroll
      for (int db = 0; db < Gm::DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[db][r] *= a;
      m = mn;
    }
    const float mm = (m == -INFINITY ? 0.0f : m) - kLog2UpFwd<T>;
    float sum = 0.0f;
#pragma unroll
    for (int jb = 0; jb < JB; ++jb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[jb][r] = __builtin_amdgcn_exp2f(fmaf(s[jb][r], p.c, -mm));
        sum += s[jb][r];
      }
    l += sum;
#pragma unroll
    for (int jb = 0; jb < JB; ++jb)
#pragma unroll
      for (int c = 0; c < Gm::PB; ++c) {
        const frag_t<T> pf = pack<T>(s[jb], c);
#pragma unroll
        for (int db = 0; db < Gm::DB; ++db)
          acc[db] = mma(lds_cols<T, DH>(vt, (wk * JB + jb) * 32 + c * Gm::KC, db, lane), pf, acc[db]);
      }
    __builtin_amdgcn_s_setprio(0);
    if (NBUF == 1) __syncthreads();
    if (tn < t_end) {
      if (NBUF == 2) buf ^= 1;
      ks.template clear<NW>(wn);
      vs.template clear<NW>(wn);
      ks.put(smem + buf * 2 * TILE);
      vs.put(smem + buf * 2 * TILE + TILE);
    }
    __syncthreads();
    t = tn;
#pragma unroll
    for (int i = 0; i < NW; ++i) w[i] = wn[i];
  }

  l = other_half_sum(l);

  if constexpr (WK > 1) {
    // acc, m and l of the WK waves that hold the same 32 rows, to LDS; the first joins them.
    __syncthreads();
    float* mine = (float*)smem + wave * 32 * DH;
#pragma unroll
    for (int db = 0; db < Gm::DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) mine[(db * 16 + r) * 64 + lane] = acc[db][r];
    if (half == 0) {
      wave_stat[wave * 64 + lane] = m;
      wave_stat[wave * 64 + 32 + lane] = l;
    }
    __syncthreads();
    if (wk > 0) return;
    float top = m;
#pragma unroll
    for (int x = 1; x < WK; ++x) top = fmaxf(top, wave_stat[(wr + x * WR) * 64 + (lane & 31)]);
    const float mm = top == -INFINITY ? 0.0f : top;
    float wt[WK], sum = 0.0f;
#pragma unroll
    for (int x = 0; x < WK; ++x) {
      wt[x] = __builtin_amdgcn_exp2f(wave_stat[(wr + x * WR) * 64 + (lane & 31)] - mm);
      sum += wt[x] * wave_stat[(wr + x * WR) * 64 + 32 + (lane & 31)];
    }
#pragma unroll
    for (int db = 0; db < Gm::DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float a = 0.0f;
#pragma unroll
        for (int x = 0; x < WK; ++x) a += wt[x] * ((const float*)smem)[(wr + x * WR) * 32 * DH + (db * 16 + r) * 64 + lane];
        acc[db][r] = a;
      }
    m = top;
    l = sum;
  }
  if (!row.in) return;
  const bool none = l == 0.0f;
  const float inv = none ? 0.0f : 1.0f / l;
  const float lse = none ? -INFINITY : m + __builtin_amdgcn_logf(l * kDownFwd<T>);
  if constexpr (SPLIT) {
    const int64_t to = ((int64_t)bh * p.splits + split) * p.R + r0 + wr * 32 + (lane & 31);
    store_col<float, Gm::DB>(p.part + to * p.D, acc, inv, half, p.D);
    if (half == 0) p.part_lse[to] = lse;
  } else {
    const int64_t h = hk * p.G + row.g;
    store_col<T, Gm::DB>((T*)p.out + b * p.so.b + h * p.so.h + row.i * p.so.s, acc, inv, half, p.D);
    if (half == 0 && p.lse != nullptr) p.lse[((int64_t)b * p.Hq + h) * p.Sq + row.i] = lse;
  }
}

// The splits of a row joined: weights exp2(lse_s - max), one lane per split, then two columns per lane.
// A wave per row, eight splits' loads in flight; latency is all it costs (64 splits of 40 rows, 8 key
// heads of 128: 6.6 us, 18.8 with one load at a time).
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
  for (int s0 = 0; s0 < p.splits; s0 += 8) {
    float2 v[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) v[x] = *(const float2*)(src + (int64_t)min(s0 + x, p.splits - 1) * p.R * p.D);
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const bool in = s0 + x < p.splits;
      const float f = lane_f(wt, (s0 + x) & 63);
      a0 = in ? fmaf(f, v[x].x, a0) : a0;
      a1 = in ? fmaf(f, v[x].y, a1) : a1;
    }
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
// In fp16 each column of ds (one row's in the dq kernel, one key's in the dk kernel) is multiplied by a
// power of two that puts its largest value so far near 2^10; when a tile passes 2^14 the column's sums
// are rescaled. Other types need no such factor.
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

// Sums of the waves of a workgroup that hold the same rows (or keys) added in order, through LDS, into
// the first's. Wave w's place in it is `mine` of `step` apart, N in all; every wave calls it.
template <int DB, int N>
__device__ __forceinline__ void join_sums(f32x16 (&acc)[DB], char* smem, int wave, int step, bool first) {
  const int lane = threadIdx.x & 63;
  float* mine = (float*)smem + wave * DB * 1024;
  __syncthreads();
  if (!first)
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) mine[(db * 16 + r) * 64 + lane] = acc[db][r];
  __syncthreads();
  if (first)
#pragma unroll
    for (int x = 1; x < N; ++x)
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[db][r] += mine[x * step * DB * 1024 + (db * 16 + r) * 64 + lane];
}

// dq, and delta for the next kernel. WR x WK = 4 waves, rows and tiles as in the forward; a row's waves
// add their dq at the end.
// The scores come again from q and k rather than from memory: at 12 heads of 8192 x 8192 they would be
// 1.6 GB to write and read. There it takes 355 us, 870 TFLOP/s, products and vector work overlapping as
// in the forward; 32 x 12 heads of 256 x 256, padded, 24 us.
template <typename T, int DH, int WR, int WK, int JB>
__global__ __launch_bounds__(kThreads, sizeof(T) * DH <= 256 ? 2 : 1) void attn_dq_kernel(Params p) {
  typedef Geo<T, DH> Gm;
  constexpr int BK = 32 * JB * WK, NW = JB * WK, TILE = BK * Gm::ROW, RB = 32 * WR;
  static_assert(WR * WK * 64 == kThreads && (WK == 1 || 4 * TILE >= kThreads / 2 * DH * 4), "joining waves reuse the tiles");
  __shared__ __attribute__((aligned(16))) char smem[4 * TILE];
  __shared__ float wave_sums[WK > 1 ? kThreads : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int wr = wave % WR, wk = wave / WR;
  const int row_tiles = (p.R + RB - 1) / RB;
  const Place at = place_of(blockIdx.x, p.B * p.Hk, row_tiles, p.causal);
  const int bh = at.pair, tile = row_tiles - 1 - at.tile;
  const int b = bh / p.Hk, hk = bh % p.Hk;
  const int r0 = tile * RB;
  int i_lo, i_hi;
  pos_range(p, r0, r0 + RB, &i_lo, &i_hi);
  const int off = p.Sk - p.Sq;
  const int kend = p.causal ? max(0, min(p.Sk, i_hi + off + 1)) : p.Sk;
  const int t_end = (kend + BK - 1) / BK;

  Row row;
  frag_t<T> qf[Gm::NC], gf[Gm::NC];
  float lse, delta;
  {
    row = row_of(p, r0 + wr * 32 + (lane & 31));
    const int64_t h = hk * p.G + row.g;
    load_row<T, DH>(qf, (const T*)p.q + b * p.sq.b + h * p.sq.h + row.i * p.sq.s, half, p.D, true);
    load_row<T, DH>(gf, (const T*)p.dout + b * p.sdo.b + h * p.sdo.h + row.i * p.sdo.s, half, p.D, true);
    frag_t<T> of[Gm::NC];
    load_row<T, DH>(of, (const T*)p.o + b * p.so.b + h * p.so.h + row.i * p.so.s, half, p.D, true);
    float a = 0.0f;
#pragma unroll
    for (int c = 0; c < Gm::NC; ++c)
#pragma unroll
      for (int e = 0; e < Gm::EPC; ++e) a += to_f32(gf[c][e]) * to_f32(of[c][e]);
    delta = other_half_sum(a);
    const int64_t to = ((int64_t)b * p.Hq + h) * p.Sq + row.i;
    lse = p.lse[to];
    if (!row.in || lse == -INFINITY) lse = INFINITY;  // exp2(s - lse) = 0
    if (half == 0 && wk == 0 && row.in) p.delta[to] = delta;
  }
  const T* kb = (const T*)p.k + b * p.sk.b + hk * p.sk.h;
  const T* vb = (const T*)p.v + b * p.sv.b + hk * p.sv.h;
  f32x16 acc[Gm::DB];
  ColScale<T> cs;
#pragma unroll
  for (int db = 0; db < Gm::DB; ++db) acc[db] = zero16();

  Stage<T, DH, BK, kThreads> ks, vs;
  ks.init(kb, p.sk.s, p.Sk, p.D);
  vs.init(vb, p.sv.s, p.Sk, p.D);
  ks.get(0);
  vs.get(0);
  KeyBits bits;
  bits.init(p, b, kend);
  uint32_t w[NW], wn[NW];
  int t = bits.next<NW>(-1, t_end, w);
  if (t < t_end) {
    if (t != 0) {
      ks.get(t * BK);
      vs.get(t * BK);
    }
    ks.template clear<NW>(w);
    vs.template clear<NW>(w);
    ks.put(smem);
    vs.put(smem + TILE);
    __syncthreads();
  }
  // In 16 bits do . o has the output's rounding in it. Where a row sees few keys delta takes most of each
  // do . v away, and that error with it (rows of up to 32 causal keys: dq off by twice its other roundings).
  // A row whose keys all lie in its first tile gets delta = sum_j p_ij (do_i . v_j) instead, which has none.
  if constexpr (sizeof(T) == 2) {
    if (t < t_end) {
      const bool last = bits.last<NW>(t, t_end);
      const int seen = (t + 1) * BK - off;  // with `causal`, rows before it see no key behind this tile
      if (last || (p.causal && i_lo < seen)) {
        float a = 0.0f;
#pragma unroll
        for (int jb = 0; jb < JB; ++jb) {
          f32x16 s = zero16(), dp = zero16();
#pragma unroll
          for (int c = 0; c < Gm::NC; ++c) {
            const int at = lds_at<T, DH>((wk * JB + jb) * 32 + (lane & 31), 2 * c + half);
            s = mma(lds_frag<T>(smem + at), qf[c], s);
            dp = mma(lds_frag<T>(smem + TILE + at), gf[c], dp);
          }
          uint32_t word = w[jb];
#pragma unroll
          for (int x = 1; x < WK; ++x) word = wk == x ? w[x * JB + jb] : word;
          word >>= 4 * half;
          const int lim = p.causal ? row.i + off - (t * BK + (wk * JB + jb) * 32 + 4 * half) : 31;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float e = __builtin_amdgcn_exp2f(fmaf(s[r], p.c, -lse));
            a = fmaf((word >> reg_row(r)) & 1 && reg_row(r) <= lim ? e : 0.0f, dp[r], a);
          }
        }
        a = other_half_sum(a);
        if constexpr (WK > 1) {
          wave_sums[wave * 64 + lane] = a;
          __syncthreads();
          a = 0.0f;
#pragma unroll
          for (int x = 0; x < WK; ++x) a += wave_sums[(wr + x * WR) * 64 + lane];
        }
        if (last || row.i < seen) {
          delta = a;
          if (half == 0 && wk == 0 && row.in) p.delta[((int64_t)b * p.Hq + hk * p.G + row.g) * p.Sq + row.i] = a;
        }
      }
    }
  }
  int buf = 0;
  while (t < t_end) {
    const int tn = bits.next<NW>(t, t_end, wn);
    if (tn < t_end) {
      ks.get(tn * BK);
      vs.get(tn * BK);
    }
    const char* kt = smem + buf * 2 * TILE;
    const char* vt = kt + TILE;
#pragma unroll
    for (int jb = 0; jb < JB; ++jb) {
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int c = 0; c < Gm::NC; ++c) {
        const int at = lds_at<T, DH>((wk * JB + jb) * 32 + (lane & 31), 2 * c + half);
        const frag_t<T> kf = lds_frag<T>(kt + at), vf = lds_frag<T>(vt + at);
        s = mma(kf, qf[c], s);
        dp = mma(vf, gf[c], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], p.c, -lse));
      uint32_t word = w[jb];
#pragma unroll
      for (int x = 1; x < WK; ++x) word = wk == x ? w[x * JB + jb] : word;
      if (word != 0xffffffffu) {
        const uint32_t mine = word >> (4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = (mine >> reg_row(r)) & 1 ? s[r] : 0.0f;
      }
      const int j0 = t * BK + (wk * JB + jb) * 32;
      if (p.causal && j0 + 31 > i_lo + off) {
        const int lim = row.i + off - (j0 + 4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = reg_row(r) <= lim ? s[r] : 0.0f;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] *= dp[r] - delta;
      cs.template apply<Gm::DB>(s, acc);
#pragma unroll
      for (int c = 0; c < Gm::PB; ++c) {
        const frag_t<T> df = pack<T>(s, c);
#pragma unroll
        for (int db = 0; db < Gm::DB; ++db)
          acc[db] = mma(lds_cols<T, DH>(kt, (wk * JB + jb) * 32 + c * Gm::KC, db, lane), df, acc[db]);
      }
    }
    if (tn < t_end) {
      buf ^= 1;
      ks.template clear<NW>(wn);
      vs.template clear<NW>(wn);
      ks.put(smem + buf * 2 * TILE);
      vs.put(smem + buf * 2 * TILE + TILE);
    }
    __syncthreads();
    t = tn;
#pragma unroll
    for (int i = 0; i < NW; ++i) w[i] = wn[i];
  }
  float f = p.scale * cs.inv();
  if constexpr (WK > 1) {
#pragma unroll
    for (int db = 0; db < Gm::DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[db][r] *= f;
    f = 1.0f;
    join_sums<Gm::DB, WK>(acc, smem, wave, WR, wk == 0);
  }
  if (wk > 0 || !row.in) return;
  store_col<T, Gm::DB>((T*)p.dq + b * p.sdq.b + (int64_t)(hk * p.G + row.g) * p.sdq.h + row.i * p.sdq.s, acc, f, half, p.D);
}

// dk and dv. KG x RG = 4 waves: wave (kg, rg) holds 32 keys (K and V as right operands, in registers) and
// walks the rows of every query head of the group in tiles of 32 IB RG, of which it takes the 32 IB
// rows rg; a key's waves add their sums at the end. A key that takes no part has its own
// column throughout, which is written as zeros: no element needs the key mask here.
// A kernel of its own, so that both sums stay in registers and nothing is added by atomics: the price is
// a second pass over the scores. At 12 heads of 8192 x 8192 x 64 it takes 480 us, 860 TFLOP/s: the
// matrix unit is busy 43% of the time and the LDS 48%, of which bank conflicts are 11. Head size 128 takes
// the registers of a whole SIMD for one wave: 16 x 32 heads over 8 key heads, 512 x 512 x 128 causal and
// padded, 145 us, where the forward takes 80 and dq 104 (tiles of 32 rows in place of 64 were slower by
// a quarter). In fp32 it spills there besides, 105 to 201 registers a lane: 8 x 16 heads of 512 x 512 x 128
// take 680 us, 51 TFLOP/s, where dq takes 278 (93) and the forward 200 (86).
template <typename T, int DH, int KG, int RG, int IB>
__global__ __launch_bounds__(kThreads, sizeof(T) * DH <= 128 ? 2 : 1) void attn_dkv_kernel(Params p) {
  typedef Geo<T, DH> Gm;
  constexpr int BR = 32 * IB * RG, KB = 32 * KG, TILE = BR * Gm::ROW;
  static_assert(KG * RG * 64 == kThreads && (RG == 1 || 4 * TILE >= kThreads / 2 * DH * 4), "joining waves reuse the tiles");
  __shared__ __attribute__((aligned(16))) char smem[4 * TILE];
  __shared__ __attribute__((aligned(16))) float stat[4 * BR];  // lse, -delta of the tile's rows
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int kg = wave % KG, rg = wave / KG;
  const int key_tiles = (p.Sk + KB - 1) / KB;
  const Place at = place_of(blockIdx.x, p.B * p.Hk, key_tiles, p.causal);
  const int bh = at.pair;
  const int b = bh / p.Hk, hk = bh % p.Hk;
  const int j0 = at.tile * KB;
  const int off = p.Sk - p.Sq;

  // This workgroup's keys: which take part, and whether any does.
  const int key = j0 + kg * 32 + (lane & 31);
  bool on = key < p.Sk;
  if (p.mask != nullptr) on = key_on(p.mask, p.mask_dtype, b * p.mask_b + min(key, p.Sk - 1)) && on;
  const bool wave_any = __any(on);
  const bool wg_any = __syncthreads_or(on);

  f32x16 dk[Gm::DB], dv[Gm::DB];
  ColScale<T> cs;
#pragma unroll
  for (int db = 0; db < Gm::DB; ++db) dk[db] = dv[db] = zero16();

  // Row tiles (g, it) of the group's heads; with `causal` those whose last row sees key j0.
  const int ntile = (p.Sq + BR - 1) / BR;
  const int first = p.causal ? min(ntile, max(0, j0 - off) / BR) : 0;
  if (wg_any && first < ntile) {
    frag_t<T> kf[Gm::NC], vf[Gm::NC];
    const int64_t j = min(key, p.Sk - 1);
    load_row<T, DH>(kf, (const T*)p.k + b * p.sk.b + hk * p.sk.h + j * p.sk.s, half, p.D, on);
    load_row<T, DH>(vf, (const T*)p.v + b * p.sv.b + hk * p.sv.h + j * p.sv.s, half, p.D, on);
    Stage<T, DH, BR, kThreads> qs, gs;
    float st = 0.0f;  // threads [0, BR): lse, [BR, 2 BR): -delta of the staged rows
    const auto get = [&](int g, int it) {
      const int64_t h = hk * p.G + g;
      qs.init((const T*)p.q + b * p.sq.b + h * p.sq.h, p.sq.s, p.Sq, p.D);
      gs.init((const T*)p.dout + b * p.sdo.b + h * p.sdo.h, p.sdo.s, p.Sq, p.D);
      qs.get(it * BR);
      gs.get(it * BR);
      if (threadIdx.x < 2 * BR) {
        const int i = it * BR + (threadIdx.x & (BR - 1));
        const float* src = threadIdx.x < BR ? p.lse : p.delta;
        st = src[((int64_t)b * p.Hq + h) * p.Sq + min(i, p.Sq - 1)];  // used by put() alone: nothing waits for it here
      }
    };
    const auto put = [&](int buf, int it) {
      qs.put(smem + buf * 2 * TILE);
      gs.put(smem + buf * 2 * TILE + TILE);
      if (threadIdx.x < 2 * BR) {
        const bool in = it * BR + (int)(threadIdx.x & (BR - 1)) < p.Sq;
        stat[buf * 2 * BR + threadIdx.x] =
            threadIdx.x >= BR ? (in ? -st : 0.0f) : in && st != -INFINITY ? st - kLog2Up<T> : INFINITY;
      }
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
        for (int i = 0; i < IB; ++i) {
          const int ib = rg * IB + i;
          const float* lse = stat + buf * 2 * BR + ib * 32 + 4 * half;
          const float* del = lse + BR;
          f32x16 start;  // do . v - delta: the sums start at -delta
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 d4 = *(const f32x4*)(del + 8 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e) start[4 * q + e] = d4[e];
          }
          f32x16 s = zero16(), dp = start;
#pragma unroll
          for (int c = 0; c < Gm::NC; ++c) {
            const int at = lds_at<T, DH>(ib * 32 + (lane & 31), 2 * c + half);
            const frag_t<T> qf = lds_frag<T>(qt + at), gf = lds_frag<T>(gt + at);
            s = mma(qf, kf[c], s);
            dp = mma(gf, vf[c], dp);
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 l4 = *(const f32x4*)(lse + 8 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * q + e] = __builtin_amdgcn_exp2f(fmaf(s[4 * q + e], p.c, -l4[e]));
          }
          const int i0 = it * BR + ib * 32 + 4 * half;
          if (p.causal && it * BR + ib * 32 < j0 + KB - 1 - off) {
            const int lim = key - off - i0;  // rows from here on see the key
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = reg_row(r) >= lim ? s[r] : 0.0f;
          }
#pragma unroll
          for (int c = 0; c < Gm::PB; ++c) {
            const frag_t<T> pf = pack<T>(s, c);
#pragma unroll
            for (int db = 0; db < Gm::DB; ++db)
              dv[db] = mma(lds_cols<T, DH>(gt, ib * 32 + c * Gm::KC, db, lane), pf, dv[db]);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] *= dp[r];
          cs.template apply<Gm::DB>(s, dk);
#pragma unroll
          for (int c = 0; c < Gm::PB; ++c) {
            const frag_t<T> df = pack<T>(s, c);
#pragma unroll
            for (int db = 0; db < Gm::DB; ++db)
              dk[db] = mma(lds_cols<T, DH>(qt, ib * 32 + c * Gm::KC, db, lane), df, dk[db]);
          }
        }
      }
      if (gn < p.G) {
        buf ^= 1;
        put(buf, itn);
      }
      __syncthreads();
      g = gn;
      it = itn;
    }
  }
  const float fv = __builtin_amdgcn_exp2f(-kLog2Up<T>), fk = on ? p.scale * fv * cs.inv() : 0.0f;
  // A key that takes no part: zeros, whatever its column held.
#pragma unroll
  for (int db = 0; db < Gm::DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      dk[db][r] = on ? dk[db][r] * fk : 0.0f;
      dv[db][r] = on ? dv[db][r] * fv : 0.0f;
    }
  if constexpr (RG > 1) {
    join_sums<Gm::DB, RG>(dk, smem, wave, KG, rg == 0);
    join_sums<Gm::DB, RG>(dv, smem, wave, KG, rg == 0);
  }
  if (rg > 0 || key >= p.Sk) return;
  store_col<T, Gm::DB>((T*)p.dk + b * p.sdk.b + hk * p.sdk.h + key * p.sdk.s, dk, 1.0f, half, p.D);
  store_col<T, Gm::DB>((T*)p.dv + b * p.sdv.b + hk * p.sdv.h + key * p.sdv.s, dv, 1.0f, half, p.D);
}

// ---- launches ----------------------------------------------------------------------------
constexpr int64_t kTargetGroups = 512;  // workgroups that fill the chip twice
constexpr int64_t kFewGroups = 192;     // fewer than that: keys are split

struct FwdPlan {
  int rows;  // of a workgroup: 32 (four waves share each tile's keys), 64 (two pairs of waves do) or 128
  int splits, tiles_per_split;
  int64_t groups;
};

// Workgroups of 64 rows (or keys), whose waves share the other side and join at the end, where those of
// 128 are few: below 200 in 16 bits, in fp32, whose products take longer, below 512 (twice the CUs).
// 12 heads of 1024 x 1024, bf16, 96 groups of 128 rows: dq 26.5 us with 128, 20.3 with 64; dk and dv 27.8
// and 20.4. 4 x 12 heads of 512 x 512, 192 groups: 18.6 and 17.6, 18.6 and 18.8; 8 x 12 heads, 384 groups:
// dk and dv 27 and 33, dq and the forward not measured there. fp32, 7 x 12 heads of 181 x 181, 168 groups:
// dk and dv 34 and 23.
bool small_groups(int64_t pairs, int64_t n, int es) { return pairs * cdiv(n, 128) < (es == 4 ? kTargetGroups : 200); }

// Keys are split over workgroups where those are few and each has many tiles. In 16 bits long keys are
// rather split than walked by small groups: 4 heads of 4096 x 4096, split 34 us and 8 to join, by small
// groups 58; 12 heads of 1024 x 1024, 16 and 7, and 18.
FwdPlan fwd_plan(int64_t B, int64_t Hk, int64_t R, int64_t Sk, int64_t D, int es) {
  FwdPlan f;
  f.rows = R <= 32 ? 32 : small_groups(B * Hk, R, es) && (es == 4 || Sk <= 2048) ? 64 : 128;
  f.groups = B * Hk * cdiv(R, f.rows);
  const int64_t tiles = cdiv(Sk, f.rows == 32 ? 128 : f.rows == 64 || D <= 64 ? 64 : 32);
  const int64_t n = f.groups >= kFewGroups ? 1 : std::min<int64_t>({cdiv(kTargetGroups, std::max<int64_t>(f.groups, 1)),
                                                                    std::max<int64_t>(tiles / 4, 1), kMaxSplits});
  f.tiles_per_split = (int)cdiv(tiles, n);
  f.splits = (int)cdiv(tiles, f.tiles_per_split);
  return f;
}

size_t fwd_bytes(const FwdPlan& f, int64_t B, int64_t Hk, int64_t R, int64_t D) {
  return f.splits > 1 ? (size_t)(B * Hk * f.splits * R) * (size_t)(D + 1) * 4 : 0;
}

template <typename T, int DH, int WR, int WK, int JB, int NBUF>
void launch_fwd_rows(const FwdPlan& f, const Params& p, hipStream_t st) {
  const dim3 grid((unsigned)(f.groups * f.splits)), block(kThreads);
  // fp32 has workgroups of 128 rows only where there are too many for a split.
  if constexpr (sizeof(T) == 2 || WR < 4) {
    if (f.splits > 1) {
      hipLaunchKernelGGL((attn_fwd_kernel<T, DH, WR, WK, JB, NBUF, true>), grid, block, 0, st, p);
      return;
    }
  }
  hipLaunchKernelGGL((attn_fwd_kernel<T, DH, WR, WK, JB, NBUF, false>), grid, block, 0, st, p);
}

template <typename T, int DH>
void launch_fwd(const FwdPlan& f, const Params& p, hipStream_t st) {
  constexpr int JB = DH == 128 ? 1 : 2;  // 32 or 64 keys a tile: in 16 bits what leaves a SIMD two waves' registers
  if (f.rows == 32) launch_fwd_rows<T, DH, 1, 4, 1, 1>(f, p, st);
  else if (f.rows == 128) launch_fwd_rows<T, DH, 4, 1, JB, 2>(f, p, st);
  else launch_fwd_rows<T, DH, 2, 2, 1, 2>(f, p, st);
  if (f.splits > 1)
    hipLaunchKernelGGL(attn_join_kernel<T>, dim3((unsigned)cdiv((int64_t)p.B * p.Hk * p.R, kThreads / 64)), dim3(kThreads),
                       0, st, p);
}

template <typename T, int DH>
void launch_bwd(const Params& p, hipStream_t st) {
  const int64_t bh = (int64_t)p.B * p.Hk;
  const dim3 block(kThreads);
  constexpr int JB = DH == 128 ? 1 : 2;
  if (p.R > 0) {
    if (!small_groups(bh, p.R, sizeof(T)))
      hipLaunchKernelGGL((attn_dq_kernel<T, DH, 4, 1, JB>), dim3((unsigned)(bh * cdiv(p.R, 128))), block, 0, st, p);
    else
      hipLaunchKernelGGL((attn_dq_kernel<T, DH, 2, 2, 1>), dim3((unsigned)(bh * cdiv(p.R, 64))), block, 0, st, p);
  }
  if (p.Sk > 0) {
    if (!small_groups(bh, p.Sk, sizeof(T)))
      hipLaunchKernelGGL((attn_dkv_kernel<T, DH, 4, 1, 2>), dim3((unsigned)(bh * cdiv(p.Sk, 128))), block, 0, st, p);
    else
      hipLaunchKernelGGL((attn_dkv_kernel<T, DH, 2, 2, 1>), dim3((unsigned)(bh * cdiv(p.Sk, 64))), block, 0, st, p);
  }
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
int read_desc(const sparton_attention_desc* d, const void* mask, bool bwd, Params* p, bool* empty) {
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
  // Workgroups of 128 rows, and of 128 keys for dk and dv; of 64 there are less than a thousand. Up to 32
  // packed rows are one workgroup either way.
  if (d->B * d->Hk > kMaxGroups / std::max({cdiv(G * d->Sq, 128), bwd ? cdiv(d->Sk, 128) : 1, (int64_t)1}))
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
  if (attn::read_desc(d, nullptr, false, &p, &empty) != SPARTON_OK || empty || p.R == 0 || p.Sk == 0) return 0;
  return attn::fwd_bytes(attn::fwd_plan(p.B, p.Hk, p.R, p.Sk, p.D, d->dtype == SPARTON_F32 ? 4 : 2), p.B, p.Hk, p.R, p.D);
}

SPARTON_EXPORT int sparton_attention_fwd(const sparton_attention_desc* d, const void* q, const void* k, const void* v,
                                         const void* mask, void* out, float* lse, void* workspace,
                                         size_t workspace_bytes, void* stream) {
  attn::Params p = {};
  bool empty;
  const int rc = attn::read_desc(d, mask, false, &p, &empty);
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
  if (attn::read_desc(d, nullptr, true, &p, &empty) != SPARTON_OK || empty) return 0;
  return (size_t)p.B * p.Hq * p.Sq * 4;
}

SPARTON_EXPORT int sparton_attention_bwd(const sparton_attention_desc* d, const void* q, const void* k, const void* v,
                                         const void* mask, const void* out, const float* lse, const void* d_out,
                                         void* d_q, void* d_k, void* d_v, void* workspace, size_t workspace_bytes,
                                         void* stream) {
  attn::Params p = {};
  bool empty;
  const int rc = attn::read_desc(d, mask, true, &p, &empty);
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
