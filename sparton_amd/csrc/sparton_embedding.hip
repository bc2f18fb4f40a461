// Embedding lookup with scaling, and its gradient by sorted tokens, on gfx950:
//     out[i, :] = scale table[id_i, :]
//     d table[v, :] = scale sum over i with id_i = v of d out[i, :], in ascending order of i; 0 for other rows
// An id outside [0, V) reads nothing: its row is NaN and it has no gradient. The padding id has a row and no
// gradient.
//
// Forward: one pass, bound by memory. 32 x 256 tokens of 768, bf16: 6.6 us; 16391 of 768, fp16: 13.1.
//
// Backward: the ids are sorted with their places (a place breaks ties, so the order is the same every time),
// and the sorted list is cut into chunks of kChunk entries. A wave takes a chunk and 64 vectors of 16 bytes of the
// row width, keeps the sum of the running id in fp32, and writes a table row where an id's entries end. The sum of
// an id whose entries go on in a neighbouring chunk is left in fp32 in the workspace, and a second launch adds such
// sums in order: in the first launch an id that half of the batch has is summed by as many waves as any other entries.
// The second has four waves for 256 columns of an id, whatever its chunks: all ids the same take 33 us in all at 8192 x 768
// bf16 and 123 at 65536, random ones of 30522 34 and 80. Rows without a token are zeroed by other waves of the first launch,
// so every row is written once and d table needs no clearing. No atomics: results are bitwise reproducible.
//
// The sort ranks each key among its wave's 64, then among 4 x 64 and 4 x 256, in a second launch among 32 x 1024 (all in
// LDS), and in further ones among 16 x 32768, ... (memory): a key's rank is its own place in its list and, by binary
// search, the number of keys before it in each of the others. No counts and no scans. These launches are bound by
// their chains of dependent reads, the sums by memory. Measured, sort + merge + sums + join: 8192 tokens of 30522 x 768
// bf16 7.6 + 8.0 + 14.9 + 4.8 us, 16391 of 250002 x 768 fp16 7.3 + 14.4 + 75.6 + 6.4 (the sums: 409 MB, 5.4 TB/s).

#include <algorithm>

#include "sparton_common.h"
#include "sparton_rows.h"

namespace sparton {
namespace emb {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;           // forward: vectors of a thread
constexpr int kTile = 1024;          // keys that one workgroup sorts
constexpr int kTileWays = 32;        // tiles that the first merge launch joins into one run, in LDS
constexpr int kWays = 16;            // runs that a later one joins
constexpr int kChunk = 32;           // sorted entries of a wave
constexpr int kInFlight = 8;
constexpr int kJoinWaves = 4;
constexpr int kZeroBytes = 32 << 10; // about what a wave zeroes
constexpr uint32_t kNone = 0x7fffffffu;  // key of an entry without a gradient: behind every id
constexpr int64_t kMaxD = 1 << 20;
constexpr uint64_t kMaxThreads = 1ull << 32;  // a launch holds fewer (past that, workgroups were left out)

// The id at place i, or kNone.
__device__ __forceinline__ uint32_t id_at(const void* ids, int ids_dtype, int64_t i, int64_t V) {
  if (ids_dtype == SPARTON_MASK_I64) {  // uniform
    const int64_t v = ((const int64_t*)ids)[i];
    return v >= 0 && v < V ? (uint32_t)v : kNone;
  }
  const int32_t v = ((const int32_t*)ids)[i];
  return v >= 0 && v < V ? (uint32_t)v : kNone;
}

// ---- forward ------------------------------------------------------------------------------
// Vector o of the row-major list of all rows' vectors: thread t of a workgroup takes kUnroll of them, kThreads
// apart. The workgroup's first row comes from one 64-bit division, each vector's from a 32-bit one.
template <typename T, int VE>
__global__ __launch_bounds__(kThreads) void embed_fwd_kernel(const void* __restrict__ ids, int ids_dtype,
                                                             const T* __restrict__ table, float scale,
                                                             T* __restrict__ out, int64_t N, int64_t V, int D) {
  const uint32_t nv = (uint32_t)cdiv(D, VE);
  const int64_t first = (int64_t)blockIdx.x * (kThreads * kUnroll);
  const int64_t row0 = first / nv;
  const uint32_t off0 = (uint32_t)(first - row0 * nv);
  int64_t row[kUnroll];
  int at[kUnroll];
  uint32_t id[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t o = off0 + u * kThreads + threadIdx.x, r = o / nv;
    row[u] = row0 + r;
    at[u] = min((int)((o - r * nv) * VE), D - VE);
    id[u] = row[u] < N ? id_at(ids, ids_dtype, row[u], V) : kNone;
  }
  vec_t<T, VE> v[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (id[u] != kNone) v[u] = load_any<T, VE>(table + (int64_t)id[u] * D + at[u]);
    else
#pragma unroll
      for (int e = 0; e < VE; ++e) v[u][e] = from_f32<T>(__builtin_nanf(""));
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (row[u] >= N) continue;
    vec_t<T, VE> w;
#pragma unroll
    for (int e = 0; e < VE; ++e) w[e] = from_f32<T>(scale * to_f32(v[u][e]));
    store_any<T, VE>(out + row[u] * D + at[u], w);
  }
}

// ---- sort ---------------------------------------------------------------------------------
// How many of the 2^LOG ascending keys lie before `key`, where keys equal to it do if `ties`.
template <int LOG> __device__ __forceinline__ int before(const uint32_t* keys, uint32_t key, bool ties) {
  const uint32_t edge = key + (ties ? 1u : 0u);  // keys are below 2^31
  int lo = 0;
#pragma unroll
  for (int s = LOG - 1; s >= 0; --s) lo += keys[lo + (1 << s) - 1] < edge ? 1 << s : 0;
  return lo + (keys[lo] < edge ? 1 : 0);
}

// One merge step within a workgroup: runs of 2^LOG ascending keys become runs of 4 x 2^LOG.
template <int LOG>
__device__ __forceinline__ void merge4(uint32_t& key, uint32_t& place, uint32_t* keys, uint32_t* places) {
  const int t = threadIdx.x, own = (t >> LOG) & 3, base = t & ~((4 << LOG) - 1);
  keys[t] = key;
  __syncthreads();
  int rank = t & ((1 << LOG) - 1);
#pragma unroll
  for (int d = 1; d < 4; ++d) {
    const int other = (own + d) & 3;
    rank += before<LOG>(keys + base + (other << LOG), key, other < own);
  }
  __syncthreads();
  keys[base + rank] = key;
  places[base + rank] = place;
  __syncthreads();
  key = keys[t];
  place = places[t];
  __syncthreads();
}

__global__ __launch_bounds__(kTile) void embed_sort_kernel(const void* __restrict__ ids, int ids_dtype, int N, int64_t V,
                                                           int64_t padding, uint32_t* __restrict__ keys_out,
                                                           uint32_t* __restrict__ places_out) {
  __shared__ uint32_t keys[kTile], places[kTile];
  const int t = threadIdx.x, lane = t & 63;
  const int i = blockIdx.x * kTile + t;
  uint32_t key = i < N ? id_at(ids, ids_dtype, i, V) : kNone;
  if (key == (uint64_t)padding) key = kNone;
  int rank = 0;
#pragma unroll 16
  for (int j = 0; j < 64; ++j)
    rank += (uint32_t)__builtin_amdgcn_readlane((int)key, j) < key + (lane > j ? 1u : 0u) ? 1 : 0;
  keys[(t & ~63) + rank] = key;
  places[(t & ~63) + rank] = (uint32_t)i;
  __syncthreads();
  key = keys[t];
  uint32_t place = places[t];
  __syncthreads();
  merge4<6>(key, place, keys, places);
  merge4<8>(key, place, keys, places);
  // Entries past N have the greatest key and places past every other's: they are last of the last tile.
  if (i < N) {
    keys_out[i] = key;
    places_out[i] = place;
  }
}

// The place, in its group of up to WAYS runs of `run` ascending keys each, that key i of the group goes to when the
// group becomes one run; `keys` are the group's `count`. The searches step together and read without a branch, so that
// their reads are in flight at once; what a search reads past the group's end, it reads from its last key and drops.
template <int WAYS, typename P, typename I>
__device__ __forceinline__ I merged_place(P keys, uint32_t key, I i, I count, I run) {
  const I own = i / run;
  const int lists = __builtin_amdgcn_readfirstlane((int)cdiv(count, run));  // the same for the whole workgroup
  I lo[WAYS];
#pragma unroll
  for (int w = 0; w < WAYS; ++w) lo[w] = 0;
  for (I step = run; step > 0; step >>= 1) {
#pragma unroll
    for (int w0 = 0; w0 < WAYS; w0 += 4) {
      if (w0 >= lists) continue;
#pragma unroll
      for (int w = w0; w < w0 + 4; ++w) {
        const I at = w * run + lo[w] + step - 1;
        const bool there = lo[w] + step <= run && at < count;
        lo[w] += there & (keys[min(at, count - 1)] < key + (w < own ? 1u : 0u)) ? step : 0;
      }
    }
  }
  I rank = i - own * run;
#pragma unroll
  for (int w = 0; w < WAYS; ++w) rank += w == own ? 0 : lo[w];
  return rank;
}

// Tiles: the group's keys are searched in LDS. 8192 keys: 8.0 us, searched in memory 17.5; 16391 keys: 14.4.
__global__ __launch_bounds__(kThreads) void embed_merge_tiles_kernel(const uint32_t* __restrict__ keys,
                                                                     const uint32_t* __restrict__ places, int N,
                                                                     uint32_t* __restrict__ keys_out,
                                                                     uint32_t* __restrict__ places_out) {
  __shared__ uint32_t all[kTile * kTileWays];
  const int64_t first = (int64_t)blockIdx.x * kThreads, i = first + threadIdx.x;
  const int64_t base = first / (kTile * kTileWays) * (kTile * kTileWays);
  const int count = (int)min((int64_t)kTile * kTileWays, N - base);
  // A tile is one vector a thread. All are on their way before the first is stored; past the last key, the last vector
  // again, and from the first whole four tiles past it, none.
  static_assert(kTile == 4 * kThreads, "a vector a thread");
  u32x4 v[kTileWays];
#pragma unroll
  for (int n0 = 0; n0 < kTileWays; n0 += 4)
    if (n0 * kTile < count)
#pragma unroll
      for (int n = n0; n < n0 + 4; ++n) v[n] = *(const u32x4*)(keys + base + min((n * kThreads + (int)threadIdx.x) * 4, (count - 1) & ~3));
  const uint32_t place = i < N ? places[i] : 0u;
#pragma unroll
  for (int n0 = 0; n0 < kTileWays; n0 += 4)
    if (n0 * kTile < count)
#pragma unroll
      for (int n = n0; n < n0 + 4; ++n) *(u32x4*)(all + (n * kThreads + threadIdx.x) * 4) = v[n];
  __syncthreads();
  if (i >= N) return;
  const uint32_t key = all[i - base];
  const int64_t to = base + merged_place<kTileWays, const uint32_t*, int>(all, key, (int)(i - base), count, kTile);
  keys_out[to] = key;
  places_out[to] = place;
}

// Longer runs, from memory.
__global__ __launch_bounds__(kThreads) void embed_merge_kernel(const uint32_t* __restrict__ keys,
                                                               const uint32_t* __restrict__ places, int N, int run,
                                                               uint32_t* __restrict__ keys_out,
                                                               uint32_t* __restrict__ places_out) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= N) return;
  const int64_t group = (int64_t)run * kWays, base = i / group * group;
  const int64_t to = base + merged_place<kWays, const uint32_t*, int64_t>(keys + base, keys[i], i - base, min(group, N - base), run);
  keys_out[to] = keys[i];
  places_out[to] = places[i];
}

// ---- backward -----------------------------------------------------------------------------
struct Params {
  const uint32_t *keys, *places;  // [N] ascending
  const void* dy;
  void* dw;
  float* part;  // [chunks][2][D]: what goes on from the chunk before, and into the one behind
  int N, D, chunks, cols, zero_rows;
  int64_t V;
  float scale;
};

template <typename T, int VE> __device__ __forceinline__ void put_row(T* to, const float* a, float scale) {
  vec_t<T, VE> o;
#pragma unroll
  for (int e = 0; e < VE; ++e) o[e] = from_f32<T>(scale * a[e]);
  store_any<T, VE>(to, o);
}

// Waves [0, chunks cols) sum chunks, the others zero the table rows that no entry names.
template <typename T, int VE> __global__ __launch_bounds__(kThreads) void embed_bwd_kernel(Params p) {
  const int lane = threadIdx.x & 63;
  const int64_t wave = (int64_t)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t sums = (int64_t)p.chunks * p.cols;
  if (wave >= sums) {
    const int64_t v0 = (wave - sums) * p.zero_rows;
    if (v0 >= p.V) return;
    const int64_t v = v0 + lane;
    bool hit = lane >= p.zero_rows || v >= p.V;
    if (!hit) {
      int lo = 0;
      for (int n = p.N; n > 0;) {  // first entry that is not before v
        const int half = n >> 1;
        if (p.keys[lo + half] < (uint32_t)v) {
          lo += half + 1;
          n -= half + 1;
        } else {
          n = half;
        }
      }
      hit = lo < p.N && p.keys[lo] == (uint32_t)v;
    }
    float zeros[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) zeros[e] = 0.0f;
    for (uint64_t bits = ~__ballot(hit); bits != 0; bits &= bits - 1) {
      T* row = (T*)p.dw + (v0 + __builtin_ctzll(bits)) * p.D;
      for (int at = lane * VE; at < p.D; at += 64 * VE) put_row<T, VE>(row + min(at, p.D - VE), zeros, 1.0f);
    }
    return;
  }
  const int chunk = (int)(wave / p.cols), col = (int)(wave % p.cols);
  const int want = (col * 64 + lane) * VE;
  const int at = min(want, p.D - VE);  // past the row's end: its last vector again, kept by nobody
  const bool mine = want < p.D;
  const int first = chunk * kChunk, n = min(kChunk, p.N - first);
  // Lane l holds entry l of the chunk; lane kChunk the entry before it, lane kChunk + 1 the one behind.
  const int look = lane < kChunk ? first + min(lane, n - 1) : lane == kChunk ? first - 1 : first + n;
  const bool real = look >= 0 && look < p.N;
  const uint32_t key = real ? p.keys[look] : kNone;
  const uint32_t place = real ? p.places[look] : 0u;
  const uint32_t prev = (uint32_t)__builtin_amdgcn_readlane((int)key, kChunk);
  const uint32_t next = (uint32_t)__builtin_amdgcn_readlane((int)key, kChunk + 1);
  float a[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) a[e] = 0.0f;
  bool from_before = prev == (uint32_t)__builtin_amdgcn_readlane((int)key, 0);
  for (int i0 = 0; i0 < n; i0 += kInFlight) {
    vec_t<T, VE> v[kInFlight];
#pragma unroll
    for (int j = 0; j < kInFlight; ++j) {  // past n: the last entry again
      const uint32_t row = (uint32_t)__builtin_amdgcn_readlane((int)place, min(i0 + j, n - 1));
      v[j] = load_any<T, VE>((const T*)p.dy + (int64_t)row * p.D + at);
    }
#pragma unroll
    for (int j = 0; j < kInFlight; ++j) {
      const int i = i0 + j;
      if (i >= n) break;
      const uint32_t id = (uint32_t)__builtin_amdgcn_readlane((int)key, i);
      if (id == kNone) return;  // it and all behind it have no gradient
#pragma unroll
      for (int e = 0; e < VE; ++e) a[e] += to_f32(v[j][e]);
      const uint32_t after = i + 1 < n ? (uint32_t)__builtin_amdgcn_readlane((int)key, i + 1) : next;
      const bool goes_on = i + 1 == n && after == id;
      if (after != id || goes_on) {
        if (mine) {
          if (from_before || goes_on) {
            float* to = p.part + ((int64_t)chunk * 2 + (from_before ? 0 : 1)) * p.D + at;
#pragma unroll
            for (int e = 0; e < VE; ++e) to[e] = a[e];
          } else {
            put_row<T, VE>((T*)p.dw + (int64_t)id * p.D + at, a, p.scale);
          }
        }
#pragma unroll
        for (int e = 0; e < VE; ++e) a[e] = 0.0f;
        from_before = false;
      }
    }
  }
}

// The id whose entries reach from chunk b into chunk b + 1 and began in chunk b: the sums of its chunks in
// their order, a run of them a wave, and the waves' sums in order. 256 columns a workgroup.
template <typename T> __global__ __launch_bounds__(64 * kJoinWaves) void embed_join_kernel(Params p) {
  __shared__ float sums[kJoinWaves][256];
  const int b = blockIdx.x, last = (b + 1) * kChunk - 1;
  const uint32_t id = p.keys[last];
  if (id == kNone || p.keys[last + 1] != id) return;
  const int first = b * kChunk;
  if (first > 0 && p.keys[first] == id && p.keys[first - 1] == id) return;  // it began before chunk b
  int lo = last + 1;
  for (int n = p.N - lo; n > 0;) {  // first entry behind the id's
    const int half = n >> 1;
    if (p.keys[lo + half] <= id) {
      lo += half + 1;
      n -= half + 1;
    } else {
      n = half;
    }
  }
  const int count = (lo - 1) / kChunk - b + 1;  // chunks: b's second sum, then first sums
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, seg = (count + kJoinWaves - 1) / kJoinWaves;
  const int end = min(count, (wave + 1) * seg);
  int at[4];
  float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int e = 0; e < 4; ++e) at[e] = min((int)blockIdx.y * 256 + e * 64 + lane, p.D - 1);
#pragma unroll 4
  for (int c = wave * seg; c < end; ++c) {
    const float* from = p.part + ((int64_t)(b + c) * 2 + (c == 0 ? 1 : 0)) * p.D;
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] += from[at[e]];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) sums[wave][e * 64 + lane] = a[e];
  __syncthreads();
  const int column = blockIdx.y * 256 + threadIdx.x;
  if (column >= p.D) return;
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < kJoinWaves; ++w) s += sums[w][threadIdx.x];
  ((T*)p.dw)[(int64_t)id * p.D + column] = from_f32<T>(p.scale * s);
}

// ---- launches -----------------------------------------------------------------------------
int vec_of(int64_t D, int dtype) {
  const int ve = dtype == SPARTON_F32 ? 4 : 8;
  return D < ve ? 1 : ve;
}

int zero_rows(int64_t D, int dtype) {
  const int64_t row = D * (dtype == SPARTON_F32 ? 4 : 2);
  return (int)std::max<int64_t>(1, std::min<int64_t>(64, kZeroBytes / row));
}

// Bytes of the two sets of sorted keys and places, and of the chunks' sums.
size_t list_bytes(int64_t N) { return (size_t)round_up(N * 4, 256); }
size_t part_bytes(int64_t N, int64_t D) { return (size_t)(cdiv(N, kChunk) * 2 * D * 4); }

int check(int64_t N, int64_t V, int64_t D, int dtype, int ids_dtype, bool backward) {
  if (N < 0 || V < 0 || D <= 0 || dtype < SPARTON_F32 || dtype > SPARTON_F16) return SPARTON_EINVAL;
  if (ids_dtype != SPARTON_MASK_I64 && ids_dtype != SPARTON_MASK_I32) return SPARTON_EINVAL;
  if (D > kMaxD || N > INT32_MAX - kTile || V >= (int64_t)kNone) return SPARTON_EUNSUPPORTED;
  const int64_t nv = cdiv(D, vec_of(D, dtype));
  if ((uint64_t)cdiv(N * nv, kThreads * kUnroll) * kThreads >= kMaxThreads) return SPARTON_EUNSUPPORTED;
  // The backward's launches: a wave for each run of table rows (a table of 2 TB, also refused forward), for a chunk's
  // columns, and the workgroups of the join.
  const uint64_t zeros = (uint64_t)cdiv(V, zero_rows(D, dtype)), sums = backward ? (uint64_t)(cdiv(N, kChunk) * cdiv(nv, 64)) : 0;
  if ((sums + zeros) * 64 + kThreads >= kMaxThreads) return SPARTON_EUNSUPPORTED;
  if (backward && (uint64_t)cdiv(N, kChunk) * cdiv(D, 256) * 64 * kJoinWaves >= kMaxThreads) return SPARTON_EUNSUPPORTED;
  return SPARTON_OK;
}

template <typename T, int VE>
void forward(const void* ids, int ids_dtype, const void* table, float scale, void* out, int64_t N, int64_t V, int64_t D,
             hipStream_t st) {
  const int64_t vectors = N * cdiv(D, VE);
  hipLaunchKernelGGL((embed_fwd_kernel<T, VE>), dim3((unsigned)cdiv(vectors, kThreads * kUnroll)), dim3(kThreads), 0, st,
                     ids, ids_dtype, (const T*)table, scale, (T*)out, N, V, (int)D);
}

template <typename T, int VE> void backward(const Params& p, hipStream_t st) {
  const int64_t waves = (int64_t)p.chunks * p.cols + cdiv(p.V, p.zero_rows);
  hipLaunchKernelGGL((embed_bwd_kernel<T, VE>), dim3((unsigned)cdiv(waves, kThreads / 64)), dim3(kThreads), 0, st, p);
  if (p.chunks > 1)
    hipLaunchKernelGGL((embed_join_kernel<T>), dim3((unsigned)(p.chunks - 1), (unsigned)cdiv(p.D, 256)),
                       dim3(64 * kJoinWaves), 0, st, p);
}

}  // namespace emb
}  // namespace sparton

using namespace sparton;

#define SPARTON_EXPORT extern "C" __attribute__((visibility("default")))

SPARTON_EXPORT int sparton_embedding_fwd(const void* ids, int ids_dtype, const void* table, float scale, void* out,
                                         int64_t N, int64_t V, int64_t D, int dtype, void* stream) {
  const int rc = emb::check(N, V, D, dtype, ids_dtype, false);
  if (rc != SPARTON_OK) return rc;
  if (N == 0) return SPARTON_OK;
  if (ids == nullptr || out == nullptr || (table == nullptr && V > 0)) return SPARTON_EINVAL;
  const uintptr_t es = dtype == SPARTON_F32 ? 4 : 2;
  if (!aligned(ids, ids_dtype == SPARTON_MASK_I64 ? 8 : 4) || !aligned(table, es) || !aligned(out, es))
    return SPARTON_EALIGN;
  hipStream_t st = (hipStream_t)stream;
  const bool one = emb::vec_of(D, dtype) == 1;
  if (dtype == SPARTON_BF16)
    one ? emb::forward<bf16, 1>(ids, ids_dtype, table, scale, out, N, V, D, st)
        : emb::forward<bf16, 8>(ids, ids_dtype, table, scale, out, N, V, D, st);
  else if (dtype == SPARTON_F16)
    one ? emb::forward<f16, 1>(ids, ids_dtype, table, scale, out, N, V, D, st)
        : emb::forward<f16, 8>(ids, ids_dtype, table, scale, out, N, V, D, st);
  else
    one ? emb::forward<float, 1>(ids, ids_dtype, table, scale, out, N, V, D, st)
        : emb::forward<float, 4>(ids, ids_dtype, table, scale, out, N, V, D, st);
  return (int)hipGetLastError();
}

SPARTON_EXPORT size_t sparton_embedding_workspace_bytes(int64_t N, int64_t V, int64_t D, int dtype) {
  if (emb::check(N, V, D, dtype, SPARTON_MASK_I64, true) != SPARTON_OK || N == 0) return 0;
  return 4 * emb::list_bytes(N) + emb::part_bytes(N, D);
}

SPARTON_EXPORT int sparton_embedding_bwd(const void* ids, int ids_dtype, const void* d_out, float scale, int64_t padding_idx,
                                         void* d_table, void* workspace, size_t workspace_bytes, int64_t N, int64_t V,
                                         int64_t D, int dtype, void* stream) {
  const int rc = emb::check(N, V, D, dtype, ids_dtype, true);
  if (rc != SPARTON_OK) return rc;
  if (V == 0) return SPARTON_OK;
  if (d_table == nullptr || (N > 0 && (ids == nullptr || d_out == nullptr))) return SPARTON_EINVAL;
  const uintptr_t es = dtype == SPARTON_F32 ? 4 : 2;
  if (!aligned(ids, ids_dtype == SPARTON_MASK_I64 ? 8 : 4) || !aligned(d_out, es) || !aligned(d_table, es))
    return SPARTON_EALIGN;
  hipStream_t st = (hipStream_t)stream;
  emb::Params p = {};
  if (N > 0) {
    if (workspace == nullptr || workspace_bytes < sparton_embedding_workspace_bytes(N, V, D, dtype))
      return SPARTON_EWORKSPACE;
    if (!aligned(workspace, 256)) return SPARTON_EALIGN;
    const size_t list = emb::list_bytes(N);
    uint32_t* k[2] = {(uint32_t*)workspace, (uint32_t*)((char*)workspace + list)};
    uint32_t* at[2] = {(uint32_t*)((char*)workspace + 2 * list), (uint32_t*)((char*)workspace + 3 * list)};
    p.part = (float*)((char*)workspace + 4 * list);
    hipLaunchKernelGGL(emb::embed_sort_kernel, dim3((unsigned)cdiv(N, emb::kTile)), dim3(emb::kTile), 0, st, ids,
                       ids_dtype, (int)N, V, padding_idx, k[0], at[0]);
    int in = 0;
    const dim3 grid((unsigned)cdiv(N, emb::kThreads)), block(emb::kThreads);
    for (int64_t run = emb::kTile; run < N; run *= run == emb::kTile ? emb::kTileWays : emb::kWays, in ^= 1) {
      if (run == emb::kTile)
        hipLaunchKernelGGL(emb::embed_merge_tiles_kernel, grid, block, 0, st, k[in], at[in], (int)N, k[in ^ 1], at[in ^ 1]);
      else
        hipLaunchKernelGGL(emb::embed_merge_kernel, grid, block, 0, st, k[in], at[in], (int)N, (int)run, k[in ^ 1], at[in ^ 1]);
    }
    p.keys = k[in];
    p.places = at[in];
  }
  const int ve = emb::vec_of(D, dtype);
  p.dy = d_out;
  p.dw = d_table;
  p.N = (int)N;
  p.D = (int)D;
  p.V = V;
  p.chunks = (int)cdiv(N, emb::kChunk);
  p.cols = (int)cdiv(cdiv(D, ve), 64);
  p.zero_rows = emb::zero_rows(D, dtype);
  p.scale = scale;
  if (dtype == SPARTON_BF16) ve == 1 ? emb::backward<bf16, 1>(p, st) : emb::backward<bf16, 8>(p, st);
  else if (dtype == SPARTON_F16) ve == 1 ? emb::backward<f16, 1>(p, st) : emb::backward<f16, 8>(p, st);
  else ve == 1 ? emb::backward<float, 1>(p, st) : emb::backward<float, 4>(p, st);
  return (int)hipGetLastError();
}
