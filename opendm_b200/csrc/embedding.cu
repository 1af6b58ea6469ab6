// Token embedding with scaling, and its gradient by sorted tokens.
//
//   lookup    out[t] = round(scale * W[ids[t]])
//   gradient  dW[v]  = round(scale * sum_{t: ids[t] = v} dY[t])
//
// Lookup: a gather bound by HBM (rows in, rows out) for a batch, by latency for a
// few tokens. A block takes 1024 groups of 8 elements in output order, each
// thread four of them with their loads in flight together.
//
// Gradient. The tokens are sorted by id (stable, so a row's tokens keep their
// order), then summed:
//   1. sort. Ids left out (padding, out of range) get the key `rows`, which
//      sorts last and is dropped.
//   2. sum. The sorted tokens are cut into chunks of C positions; a warp takes
//      one chunk and 256 columns and adds the rows of dY in sorted order in
//      fp32 registers, writing a row of dW where the key changes. A run of
//      equal keys that goes past its chunk is finished by the warp it starts
//      in, unless it covers the whole next chunk (a "long" run): then each
//      chunk writes its fp32 partial row and the run is put on a list.
//   3. join. Each long run's partial rows are added in chunk order.
// Every sum's order depends on the sorted tokens alone: no floating-point
// atomics, two calls give the same bits.

#include "common.cuh"
#include "internal.h"

namespace muon {

namespace {

constexpr int kVec = 8;             // elements a lane handles of a row
constexpr int kSlice = 32 * kVec;   // columns of one warp
constexpr int kMaxChunk = 32;       // sorted positions of one warp (one key per lane)
constexpr int64_t kMaxIndex = 0x7ffffffeLL;

__device__ __forceinline__ int64_t load_id(const void* ids, bool wide, int64_t t) {
  return wide ? reinterpret_cast<const int64_t*>(ids)[t] : int64_t(reinterpret_cast<const int32_t*>(ids)[t]);
}

__device__ __forceinline__ void record_error(int* err, int code) { atomicCAS(err, 0, code); }

// 8 consecutive elements as fp32.
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[kVec]) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[kVec]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[kVec]) {
  uint4 raw;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = raw;
}
__device__ __forceinline__ void store8(float* p, const float (&v)[kVec]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }

// ------------------------------------------------------------------ lookup
constexpr int LK_THREADS = 256;
constexpr int LK_PER = 4;

// `group` consecutive elements per unit: 8 (vector path) or 1.
template <typename W, typename O, bool kVector>
__global__ void __launch_bounds__(LK_THREADS) lookup_kernel(const W* __restrict__ weight, int64_t rows, int64_t ld,
                                                            const void* __restrict__ ids, bool wide, int64_t tokens,
                                                            uint32_t units, int64_t dim, float scale,
                                                            O* __restrict__ out, int* err) {
  const int64_t base = int64_t(blockIdx.x) * (LK_THREADS * LK_PER);
  const int64_t row0 = base / units;
  const uint32_t col0 = uint32_t(base - row0 * units);
  float v[LK_PER][kVector ? kVec : 1];
  int64_t dst[LK_PER];
#pragma unroll
  for (int i = 0; i < LK_PER; ++i) {
    const uint32_t c = col0 + i * LK_THREADS + threadIdx.x;
    const uint32_t over = c / units;
    const int64_t t = row0 + over;
    const int64_t col = int64_t(c - over * units) * (kVector ? kVec : 1);
    dst[i] = t < tokens ? t * dim + col : -1;
    if (t >= tokens) continue;
    const int64_t id = load_id(ids, wide, t);
    if (id < 0 || id >= rows) {
#pragma unroll
      for (int k = 0; k < (kVector ? kVec : 1); ++k) v[i][k] = 0.f;
      if (col == 0) record_error(err, MUON_DEV_BAD_INDEX);
    } else if constexpr (kVector) {
      load8(weight + id * ld + col, v[i]);
    } else {
      v[i][0] = load1(weight + id * ld + col);
    }
  }
#pragma unroll
  for (int i = 0; i < LK_PER; ++i) {
    if (dst[i] < 0) continue;
#pragma unroll
    for (int k = 0; k < (kVector ? kVec : 1); ++k) v[i][k] *= scale;
    if constexpr (kVector)
      store8(out + dst[i], v[i]);
    else
      store1(out + dst[i], v[i][0]);
  }
}

template <typename W, typename O>
int run_lookup(const void* weight, int64_t rows, int64_t dim, int64_t ld, const void* ids, bool wide, int64_t tokens,
               float scale, void* out, int* err, cudaStream_t stream) {
  const bool vec = dim % kVec == 0 && ld % kVec == 0 &&
                   ((reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
  const int64_t units = vec ? dim / kVec : dim;
  const int64_t blocks = (tokens * units + LK_THREADS * LK_PER - 1) / (LK_THREADS * LK_PER);
  if (blocks > 0x7fffffffLL) return set_error(MUON_ERR_ARG, "embedding output too large");
  const unsigned grid = static_cast<unsigned>(blocks);
  if (vec)
    lookup_kernel<W, O, true><<<grid, LK_THREADS, 0, stream>>>(static_cast<const W*>(weight), rows, ld, ids, wide,
                                                               tokens, static_cast<uint32_t>(units), dim, scale,
                                                               static_cast<O*>(out), err);
  else
    lookup_kernel<W, O, false><<<grid, LK_THREADS, 0, stream>>>(static_cast<const W*>(weight), rows, ld, ids, wide,
                                                                tokens, static_cast<uint32_t>(units), dim, scale,
                                                                static_cast<O*>(out), err);
  return check_cuda(cudaGetLastError(), "embedding launch");
}

// -------------------------------------------------------------------- sort
// Least-significant-digit radix sort of (key, position), digits of at most 9
// bits: 2 passes for vocabularies below 2^18. A pass is three launches: digit
// counts per tile, their scan, and the stable scatter.
constexpr int RS_THREADS = 256;
constexpr int RS_WARPS = RS_THREADS / 32;
constexpr int RS_PER = 8;
constexpr int RS_TILE = RS_THREADS * RS_PER;
constexpr int RS_BITS = 9;
constexpr int RS_BINS = 1 << RS_BITS;

struct SortSource {
  const void* ids;  // pass 0: token ids
  bool wide;
  int64_t rows;
  int64_t padding;
  const uint32_t* keys;  // later passes
  const uint32_t* pos;
};

// Key of token t: its id, or `rows` when it takes no part.
__device__ __forceinline__ uint32_t token_key(const SortSource& s, int64_t t, int* err) {
  const int64_t id = load_id(s.ids, s.wide, t);
  if (id < 0 || id >= s.rows) {
    if (err) record_error(err, MUON_DEV_BAD_INDEX);
    return static_cast<uint32_t>(s.rows);
  }
  return id == s.padding ? static_cast<uint32_t>(s.rows) : static_cast<uint32_t>(id);
}

__global__ void __launch_bounds__(RS_THREADS) radix_count_kernel(SortSource s, int64_t n, int shift, int bits,
                                                                 uint32_t* __restrict__ hist, uint32_t* long_count,
                                                                 int* err) {
  __shared__ uint32_t h[RS_BINS];
  const int bins = 1 << bits;
  for (int b = threadIdx.x; b < bins; b += RS_THREADS) h[b] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *long_count = 0;
  __syncthreads();
  const int64_t base = int64_t(blockIdx.x) * RS_TILE;
#pragma unroll
  for (int i = 0; i < RS_PER; ++i) {
    const int64_t t = base + i * RS_THREADS + threadIdx.x;
    if (t < n) {
      const uint32_t key = s.keys ? s.keys[t] : token_key(s, t, err);
      atomicAdd(&h[(key >> shift) & (bins - 1)], 1u);
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += RS_THREADS) hist[int64_t(blockIdx.x) * RS_BINS + b] = h[b];
}

// hist[tile][bin] -> first output position of that tile's keys of that bin.
__global__ void __launch_bounds__(RS_BINS) radix_scan_kernel(uint32_t* __restrict__ hist, int64_t tiles, int bits) {
  __shared__ uint32_t warp_sum[RS_BINS / 32];
  const int bin = threadIdx.x, bins = 1 << bits, lane = bin & 31, warp = bin >> 5;
  uint32_t total = 0;
  if (bin < bins)
    for (int64_t t = 0; t < tiles; ++t) total += hist[t * RS_BINS + bin];
  uint32_t inc = total;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += up;
  }
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  uint32_t run = inc - total;
  for (int w = 0; w < warp; ++w) run += warp_sum[w];
  if (bin < bins)
    for (int64_t t = 0; t < tiles; ++t) {
      const uint32_t c = hist[t * RS_BINS + bin];
      hist[t * RS_BINS + bin] = run;
      run += c;
    }
}

__global__ void __launch_bounds__(RS_THREADS) radix_scatter_kernel(SortSource s, int64_t n, int shift, int bits,
                                                                   const uint32_t* __restrict__ first,
                                                                   uint32_t* __restrict__ out_keys,
                                                                   uint32_t* __restrict__ out_pos) {
  __shared__ uint32_t h[RS_WARPS][RS_BINS];
  const int bins = 1 << bits, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int b = lane; b < bins; b += 32) h[warp][b] = 0;
  __syncwarp();
  const int64_t base = int64_t(blockIdx.x) * RS_TILE + warp * (32 * RS_PER) + lane;
  uint32_t key[RS_PER], pos[RS_PER], rank[RS_PER];
#pragma unroll
  for (int i = 0; i < RS_PER; ++i) {
    const int64_t t = base + i * 32;
    if (t < n) {
      key[i] = s.keys ? s.keys[t] : token_key(s, t, nullptr);
      pos[i] = s.keys ? s.pos[t] : static_cast<uint32_t>(t);
    }
  }
#pragma unroll
  for (int i = 0; i < RS_PER; ++i) {
    const bool in = base + i * 32 < n;
    const uint32_t d = in ? (key[i] >> shift) & (bins - 1) : 0xffffffffu;
    const uint32_t peers = __match_any_sync(0xffffffffu, d);
    const uint32_t before = __popc(peers & ((1u << lane) - 1u));
    uint32_t count = 0;
    if (in) count = h[warp][d];
    __syncwarp();
    if (in && before == 0) h[warp][d] = count + __popc(peers);
    __syncwarp();
    rank[i] = count + before;
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += RS_THREADS) {
    uint32_t run = first[int64_t(blockIdx.x) * RS_BINS + b];
#pragma unroll
    for (int w = 0; w < RS_WARPS; ++w) {
      const uint32_t c = h[w][b];
      h[w][b] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RS_PER; ++i) {
    if (base + i * 32 >= n) continue;
    const uint32_t to = h[warp][(key[i] >> shift) & (bins - 1)] + rank[i];
    out_keys[to] = key[i];
    out_pos[to] = pos[i];
  }
}

// ------------------------------------------------------------------- heads
// Row form: how many runs start before each chunk. chunk_base[c] counts the
// run starts between the chunk's tile of HD_TILE positions and the chunk;
// tile_heads[t] the run starts in tile t.
constexpr int HD_THREADS = 256;
constexpr int HD_TILE = 4096;

__global__ void __launch_bounds__(HD_THREADS) heads_kernel(const uint32_t* __restrict__ keys, int64_t n,
                                                           uint32_t rows, int chunk, uint32_t* __restrict__ chunk_base,
                                                           uint32_t* __restrict__ tile_heads) {
  constexpr int kPer = HD_TILE / HD_THREADS;  // consecutive positions per thread
  __shared__ uint32_t warp_sum[HD_THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t base = int64_t(blockIdx.x) * HD_TILE + int64_t(threadIdx.x) * kPer;
  uint32_t flags = 0;
  uint32_t prev = base > 0 && base < n ? keys[base - 1] : 0xffffffffu;
  for (int i = 0; i < kPer && base + i < n; ++i) {
    const uint32_t k = keys[base + i];
    if (k != prev && k < rows) flags |= 1u << i;
    prev = k;
  }
  const uint32_t mine = __popc(flags);
  uint32_t inc = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += up;
  }
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  uint32_t before = inc - mine;
  for (int w = 0; w < warp; ++w) before += warp_sum[w];
  for (int i = 0; i < kPer; ++i)
    if (base + i < n && (base + i) % chunk == 0)
      chunk_base[(base + i) / chunk] = before + __popc(flags & ((1u << i) - 1u));
  if (threadIdx.x == HD_THREADS - 1) tile_heads[blockIdx.x] = before + mine;
}

// --------------------------------------------------------------------- sum
constexpr int SUM_THREADS = 256;
constexpr int SUM_WARPS = SUM_THREADS / 32;

template <bool kVector, typename T>
__device__ __forceinline__ void load_cols(const T* row, int64_t col, int64_t dim, int lane, float (&v)[kVec]) {
  if constexpr (kVector) {
    if (col < dim) {
      load8(row + col, v);
    } else {
#pragma unroll
      for (int k = 0; k < kVec; ++k) v[k] = 0.f;
    }
  } else {
#pragma unroll
    for (int k = 0; k < kVec; ++k) v[k] = col + 32 * k < dim ? load1(row + col + 32 * k) : 0.f;
  }
}

template <bool kVector, typename T>
__device__ __forceinline__ void store_cols(T* row, int64_t col, int64_t dim, const float (&v)[kVec]) {
  if constexpr (kVector) {
    if (col < dim) store8(row + col, v);
  } else {
#pragma unroll
    for (int k = 0; k < kVec; ++k)
      if (col + 32 * k < dim) store1(row + col + 32 * k, v[k]);
  }
}

struct SumArgs {
  const uint32_t* keys;
  const uint32_t* pos;
  int64_t n;
  int64_t rows;
  int64_t dim;
  int chunk;
  int64_t chunks;
  int64_t slices;
  float scale;
  const uint32_t* chunk_base;  // row form
  const uint32_t* tile_heads;
  int64_t cap;
  int64_t* out_ids;  // NULL: dense form
  int64_t* count;
  float* partial;  // [chunks][2][slices * kSlice]: a run from an earlier chunk; a long run starting here
  uint32_t* long_list;
  uint32_t* long_count;
};

template <typename G, typename O, bool kVector>
__global__ void __launch_bounds__(SUM_THREADS) sum_kernel(const G* __restrict__ grad, O* __restrict__ out, SumArgs a) {
  constexpr int kUnroll = sizeof(G) == 2 ? 8 : 4;
  __shared__ uint32_t red[2][SUM_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t unit = int64_t(blockIdx.x) * SUM_WARPS + warp;
  const int64_t c = unit / a.slices;
  const int64_t slice = unit - c * a.slices;
  const int64_t s0 = c * a.chunk;
  uint32_t slot = 0, total = 0;
  if (a.out_ids) {
    // distinct rows before this block's first tile, and in all
    const int64_t tile0 = (int64_t(blockIdx.x) * SUM_WARPS / a.slices) * a.chunk / HD_TILE;
    const int64_t tiles = (a.n + HD_TILE - 1) / HD_TILE;
    uint32_t low = 0, all = 0;
    for (int64_t t = threadIdx.x; t < tiles; t += SUM_THREADS) {
      const uint32_t h = a.tile_heads[t];
      all += h;
      if (t < tile0) low += h;
    }
    low = __reduce_add_sync(0xffffffffu, low);
    all = __reduce_add_sync(0xffffffffu, all);
    if (lane == 0) red[0][warp] = low, red[1][warp] = all;
    __syncthreads();
    for (int w = 0; w < SUM_WARPS; ++w) slot += red[0][w], total += red[1][w];
    if (c < a.chunks) {
      for (int64_t t = tile0; t < s0 / HD_TILE; ++t) slot += a.tile_heads[t];
      slot += a.chunk_base[c];
    }
    if (unit == 0 && lane == 0) *a.count = total;
  }
  if (c >= a.chunks) return;
  const int len = static_cast<int>(min(int64_t(a.chunk), a.n - s0));
  const int64_t col = slice * kSlice + (kVector ? lane * kVec : lane);
  const uint32_t none = 0xffffffffu;
  // keys and positions of this chunk and the next, one per lane each
  const uint32_t dropped = static_cast<uint32_t>(a.rows);
  const int64_t s1 = s0 + len;
  uint32_t key_a = lane < len ? a.keys[s0 + lane] : none;
  uint32_t pos_a = lane < len ? a.pos[s0 + lane] : 0;
  const int next = static_cast<int>(min(int64_t(a.chunk), a.n - s1));
  uint32_t key_b = lane < next ? a.keys[s1 + lane] : none;
  uint32_t pos_b = lane < next ? a.pos[s1 + lane] : 0;
  if (a.out_ids) {  // this chunk's share of the rows past the count
    float zero[kVec] = {};
    for (int i = 0; i < a.chunk; ++i) {
      const int64_t r = s0 + i;
      if (r >= int64_t(total) && r < a.cap) {
        store_cols<kVector>(out + r * a.dim, col, a.dim, zero);
        if (slice == 0 && lane == 0) a.out_ids[r] = 0;
      }
    }
  }
  const uint32_t first = __shfl_sync(0xffffffffu, key_a, 0);
  const uint32_t last = __shfl_sync(0xffffffffu, key_a, len - 1);
  const uint32_t before = s0 > 0 ? a.keys[s0 - 1] : none;
  const bool whole = len == a.chunk && first == last;
  int begin = 0;           // first position this warp adds
  bool lead_partial = false;  // ... belonging to a long run of an earlier chunk
  if (s0 > 0 && before == first) {
    const bool starts_before_last = s0 - a.chunk > 0 && a.keys[s0 - a.chunk - 1] == first;
    if (whole || starts_before_last)
      lead_partial = true;
    else  // the warp of the chunk before finishes this run
      begin = __popc(__ballot_sync(0xffffffffu, key_a == first));
  }
  // end of the rows this warp adds: the chunk, plus the rest of a run that does not cover the next chunk
  int end = len;
  bool tail_partial = false;
  const uint32_t next_first = __shfl_sync(0xffffffffu, key_b, 0);
  if (begin < len && next > 0 && next_first == last) {
    const bool from_here = !(lead_partial && whole);  // the last run starts in this chunk
    const bool next_whole = next == a.chunk && __shfl_sync(0xffffffffu, key_b, a.chunk - 1) == last;
    if (next_whole)
      tail_partial = from_here;
    else if (from_here)
      end = len + __popc(__ballot_sync(0xffffffffu, key_b == last));
  }
  if (tail_partial && slice == 0 && lane == 0 && last != dropped) a.long_list[atomicAdd(a.long_count, 1u)] = uint32_t(c);
  const int64_t pitch = a.slices * kSlice;
  float* part = a.partial + c * 2 * pitch;
  float acc[kVec] = {};
  for (int r0 = begin; r0 < end; r0 += kUnroll) {
    float v[kUnroll][kVec];
    uint32_t k[kUnroll + 1];
#pragma unroll
    for (int i = 0; i <= kUnroll; ++i) {
      const int r = r0 + i;
      const bool in_b = r >= len;
      const uint32_t ka = __shfl_sync(0xffffffffu, key_a, r & 31), kb = __shfl_sync(0xffffffffu, key_b, (r - len) & 31);
      k[i] = in_b ? (r - len < next ? kb : none) : ka;
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int r = r0 + i;
      const uint32_t pa = __shfl_sync(0xffffffffu, pos_a, r & 31), pb = __shfl_sync(0xffffffffu, pos_b, (r - len) & 31);
      if (r < end && k[i] != dropped) load_cols<kVector>(grad + int64_t(r < len ? pa : pb) * a.dim, col, a.dim, lane, v[i]);
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int r = r0 + i;
      if (r >= end || k[i] == dropped) continue;
#pragma unroll
      for (int j = 0; j < kVec; ++j) acc[j] += v[i][j];
      const bool run_ends = k[i + 1] != k[i];
      if (!run_ends && r + 1 < end) continue;
      if (lead_partial && k[i] == first) {
        store_cols<true>(part, slice * kSlice + lane * kVec, pitch, acc);
      } else if (tail_partial && k[i] == last) {
        store_cols<true>(part + pitch, slice * kSlice + lane * kVec, pitch, acc);
        ++slot;
      } else {
        float w[kVec];
#pragma unroll
        for (int j = 0; j < kVec; ++j) w[j] = acc[j] * a.scale;
        const int64_t row = a.out_ids ? int64_t(slot) : int64_t(k[i]);
        store_cols<kVector>(out + row * a.dim, col, a.dim, w);
        if (a.out_ids && slice == 0 && lane == 0) a.out_ids[slot] = k[i];
        ++slot;
      }
#pragma unroll
      for (int j = 0; j < kVec; ++j) acc[j] = 0.f;
    }
  }
}

// -------------------------------------------------------------------- join
// One block per (long run, slice): the run's partial rows, split evenly over
// the warps in chunk order, then the warps' sums in order.
template <typename O, bool kVector>
__global__ void __launch_bounds__(SUM_THREADS) join_kernel(O* __restrict__ out, SumArgs a) {
  __shared__ float red[SUM_WARPS][kSlice];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t pitch = a.slices * kSlice;
  const int64_t jobs = int64_t(*a.long_count) * a.slices;
  for (int64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
    const int64_t c0 = a.long_list[job / a.slices];
    const int64_t slice = job % a.slices;
    const uint32_t key = a.keys[(c0 + 1) * a.chunk];
    // last chunk the run reaches: the last c1 whose first key is the run's
    int64_t lo = c0 + 1, hi = a.chunks - 1;
    while (lo < hi) {
      const int64_t mid = (lo + hi + 1) >> 1;
      if (a.keys[mid * a.chunk] == key)
        lo = mid;
      else
        hi = mid - 1;
    }
    const int64_t n_parts = lo - c0 + 1;
    const int64_t per = (n_parts + SUM_WARPS - 1) / SUM_WARPS;
    const int64_t p0 = min(n_parts, warp * per), p1 = min(n_parts, p0 + per);
    float acc[kVec] = {};
    const int64_t off = slice * kSlice + lane * kVec;
    for (int64_t p = p0; p < p1; ++p) {
      float v[kVec];
      load8(a.partial + ((c0 + p) * 2 + (p == 0 ? 1 : 0)) * pitch + off, v);
#pragma unroll
      for (int j = 0; j < kVec; ++j) acc[j] += v[j];
    }
    store8(&red[warp][lane * kVec], acc);
    __syncthreads();
    if (warp == 0) {
      int64_t row = key;
      if (a.out_ids) {
        // the run's row: runs starting before chunk c0's end, less one
        const int64_t tile = c0 * a.chunk / HD_TILE;
        uint32_t slot = 0;
        for (int64_t t = lane; t < tile; t += 32) slot += a.tile_heads[t];
        slot = __reduce_add_sync(0xffffffffu, slot) + a.chunk_base[c0];
        // run starts inside chunk c0
        const int64_t s = c0 * a.chunk + lane;
        const bool head = lane < a.chunk && (s == 0 || a.keys[s - 1] != a.keys[s]);
        row = int64_t(slot) + __popc(__ballot_sync(0xffffffffu, head)) - 1;
        if (slice == 0 && lane == 0) a.out_ids[row] = key;
      }
      // element j of this lane sits at column lane * 8 + j (vector) or lane + 32 j of the slice, in both
      // layouts at red[..][lane * 8 + j]
      float w[kVec];
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        float sum = 0.f;
        for (int q = 0; q < SUM_WARPS; ++q) sum += red[q][lane * kVec + j];
        w[j] = sum * a.scale;
      }
      store_cols<kVector>(out + row * a.dim, slice * kSlice + (kVector ? lane * kVec : lane), a.dim, w);
    }
    __syncthreads();
  }
}

int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }

int bits_for(int64_t rows) {  // keys 0 .. rows
  int bits = 1;
  while ((int64_t(1) << bits) <= rows) ++bits;
  return bits;
}

// Chunk length: long chunks save partial rows and searches, short ones give
// more warps.
int chunk_for(int64_t tokens, int64_t slices) {
  int chunk = kMaxChunk;
  while (chunk > 8 && tokens / chunk * slices < 148 * 32) chunk /= 2;
  return chunk;
}

struct GradLayout {
  int64_t keys[2], pos[2], hist, chunk_base, tile_heads, long_list, long_count, partial, total;
  int64_t tiles, chunks, slices;
  int chunk;
};

GradLayout grad_layout(int64_t n, int64_t dim) {
  GradLayout l;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += align256(bytes);
    return here;
  };
  l.tiles = (n + RS_TILE - 1) / RS_TILE;
  l.slices = (dim + kSlice - 1) / kSlice;
  l.chunk = chunk_for(n, l.slices);
  l.chunks = (n + l.chunk - 1) / l.chunk;
  for (int i = 0; i < 2; ++i) l.keys[i] = take(4 * n), l.pos[i] = take(4 * n);
  l.hist = take(4 * l.tiles * RS_BINS);
  l.chunk_base = take(4 * l.chunks);
  l.tile_heads = take(4 * ((n + HD_TILE - 1) / HD_TILE));
  l.long_list = take(4 * l.chunks);
  l.long_count = take(4);
  l.partial = take(8 * l.chunks * l.slices * kSlice);
  l.total = at;
  return l;
}

bool float_type(int dtype) { return dtype == MUON_BF16 || dtype == MUON_F32; }

// elements x 4 bytes must fit an int64 with room to spare
bool too_large(int64_t a, int64_t b) { return b > 0 && a > (int64_t(1) << 58) / b; }

template <typename G, typename O>
int run_sum(const void* grad, void* out, const SumArgs& a, cudaStream_t stream) {
  const bool vec = a.dim % kVec == 0 &&
                   ((reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
  const int64_t blocks = (a.chunks * a.slices + SUM_WARPS - 1) / SUM_WARPS;
  if (blocks > 0x7fffffffLL) return set_error(MUON_ERR_ARG, "embedding gradient too large");
  const unsigned grid = static_cast<unsigned>(blocks);
  const G* g = static_cast<const G*>(grad);
  O* o = static_cast<O*>(out);
  if (vec)
    sum_kernel<G, O, true><<<grid, SUM_THREADS, 0, stream>>>(g, o, a);
  else
    sum_kernel<G, O, false><<<grid, SUM_THREADS, 0, stream>>>(g, o, a);
  if (check_cuda(cudaGetLastError(), "embedding gradient sum launch")) return MUON_ERR_CUDA;
  const unsigned join_grid = static_cast<unsigned>(a.chunks * a.slices < 592 ? a.chunks * a.slices : 592);
  if (vec)
    join_kernel<O, true><<<join_grid, SUM_THREADS, 0, stream>>>(o, a);
  else
    join_kernel<O, false><<<join_grid, SUM_THREADS, 0, stream>>>(o, a);
  return check_cuda(cudaGetLastError(), "embedding gradient join launch");
}

}  // namespace

int launch_embedding(const void* weight, int weight_dtype, int64_t rows, int64_t dim, int64_t ld, const void* ids,
                     int ids_dtype, int64_t tokens, float scale, void* out, int out_dtype, int* err,
                     cudaStream_t stream) {
  if (rows < 0 || dim < 0 || tokens < 0 || ld < dim) return set_error(MUON_ERR_ARG, "negative embedding size or ld < dim");
  if (!float_type(weight_dtype) || !float_type(out_dtype))
    return set_error(MUON_ERR_ARG, "embedding dtypes must be MUON_BF16 or MUON_F32");
  if (ids_dtype != MUON_I32 && ids_dtype != MUON_I64) return set_error(MUON_ERR_ARG, "ids must be MUON_I32 or MUON_I64");
  if (too_large(rows, ld) || too_large(tokens, dim) || dim >= kMaxIndex)
    return set_error(MUON_ERR_ARG, "embedding too large");
  if (tokens == 0 || dim == 0) return MUON_OK;
  if ((rows > 0 && !weight) || !ids || !out || !err) return set_error(MUON_ERR_ARG, "null embedding pointer");
  const bool wide = ids_dtype == MUON_I64, wb = weight_dtype == MUON_BF16, ob = out_dtype == MUON_BF16;
  using bf = __nv_bfloat16;
  if (wb && ob) return run_lookup<bf, bf>(weight, rows, dim, ld, ids, wide, tokens, scale, out, err, stream);
  if (wb) return run_lookup<bf, float>(weight, rows, dim, ld, ids, wide, tokens, scale, out, err, stream);
  if (ob) return run_lookup<float, bf>(weight, rows, dim, ld, ids, wide, tokens, scale, out, err, stream);
  return run_lookup<float, float>(weight, rows, dim, ld, ids, wide, tokens, scale, out, err, stream);
}

int64_t embedding_grad_workspace_bytes(int64_t tokens, int64_t rows, int64_t dim) {
  if (tokens < 0 || rows < 0 || dim < 0 || tokens >= kMaxIndex || rows >= kMaxIndex || dim >= kMaxIndex ||
      too_large(tokens, dim) || too_large(rows, dim))
    return -1;
  return tokens == 0 || dim == 0 ? 256 : grad_layout(tokens, dim).total;
}

int launch_embedding_grad(const void* grad, int grad_dtype, const void* ids, int ids_dtype, int64_t tokens,
                          int64_t rows, int64_t dim, int64_t padding_idx, float scale, void* out, int out_dtype,
                          int64_t* out_ids, int64_t* count, void* workspace, int64_t workspace_bytes, int* err,
                          cudaStream_t stream) {
  const int64_t need = embedding_grad_workspace_bytes(tokens, rows, dim);
  if (need < 0) return set_error(MUON_ERR_ARG, "embedding gradient sizes out of range");
  if (!float_type(grad_dtype) || !float_type(out_dtype))
    return set_error(MUON_ERR_ARG, "embedding gradient dtypes must be MUON_BF16 or MUON_F32");
  if (ids_dtype != MUON_I32 && ids_dtype != MUON_I64) return set_error(MUON_ERR_ARG, "ids must be MUON_I32 or MUON_I64");
  if (padding_idx != -1 && (padding_idx < 0 || padding_idx >= rows))
    return set_error(MUON_ERR_ARG, "padding_idx must be -1 or a row");
  if (out_ids && !count) return set_error(MUON_ERR_ARG, "the row form needs a count");
  const int64_t cap = tokens < rows ? tokens : rows;
  const int64_t out_rows = out_ids ? cap : rows;
  if (out_rows * dim > 0 && !out) return set_error(MUON_ERR_ARG, "null embedding gradient output");
  if (tokens > 0 && (!ids || !err || (dim > 0 && !grad))) return set_error(MUON_ERR_ARG, "null embedding gradient pointer");
  const int64_t out_bytes = rows * dim * (out_dtype == MUON_BF16 ? 2 : 4);
  if (tokens == 0 || rows == 0 || dim == 0) {
    if (out_ids) {
      if (check_cuda(cudaMemsetAsync(count, 0, sizeof(int64_t), stream), "embedding gradient count")) return MUON_ERR_CUDA;
      if (cap > 0)
        return check_cuda(cudaMemsetAsync(out_ids, 0, sizeof(int64_t) * cap, stream), "embedding gradient ids");
      return MUON_OK;
    }
    return out_bytes > 0 ? check_cuda(cudaMemsetAsync(out, 0, out_bytes, stream), "embedding gradient zeros") : MUON_OK;
  }
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
    return set_error(MUON_ERR_ARG, "embedding gradient workspace missing, too small or misaligned");
  const GradLayout l = grad_layout(tokens, dim);
  char* base = static_cast<char*>(workspace);
  auto u32 = [&](int64_t off) { return reinterpret_cast<uint32_t*>(base + off); };
  // sort
  const int bits = bits_for(rows), passes = (bits + RS_BITS - 1) / RS_BITS, per = (bits + passes - 1) / passes;
  SortSource src{ids, ids_dtype == MUON_I64, rows, padding_idx, nullptr, nullptr};
  const unsigned tiles = static_cast<unsigned>(l.tiles);
  int cur = 0;
  for (int p = 0; p < passes; ++p) {
    radix_count_kernel<<<tiles, RS_THREADS, 0, stream>>>(src, tokens, p * per, per, u32(l.hist), u32(l.long_count),
                                                         p == 0 ? err : nullptr);
    if (check_cuda(cudaGetLastError(), "radix count launch")) return MUON_ERR_CUDA;
    radix_scan_kernel<<<1, RS_BINS, 0, stream>>>(u32(l.hist), l.tiles, per);
    if (check_cuda(cudaGetLastError(), "radix scan launch")) return MUON_ERR_CUDA;
    radix_scatter_kernel<<<tiles, RS_THREADS, 0, stream>>>(src, tokens, p * per, per, u32(l.hist), u32(l.keys[cur]),
                                                           u32(l.pos[cur]));
    if (check_cuda(cudaGetLastError(), "radix scatter launch")) return MUON_ERR_CUDA;
    src.keys = u32(l.keys[cur]);
    src.pos = u32(l.pos[cur]);
    cur ^= 1;
  }
  if (out_ids) {
    const unsigned grid = static_cast<unsigned>((tokens + HD_TILE - 1) / HD_TILE);
    heads_kernel<<<grid, HD_THREADS, 0, stream>>>(src.keys, tokens, static_cast<uint32_t>(rows), l.chunk,
                                                  u32(l.chunk_base), u32(l.tile_heads));
    if (check_cuda(cudaGetLastError(), "run heads launch")) return MUON_ERR_CUDA;
  } else if (check_cuda(cudaMemsetAsync(out, 0, out_bytes, stream), "embedding gradient zeros")) {
    return MUON_ERR_CUDA;
  }
  SumArgs a{};
  a.keys = src.keys;
  a.pos = src.pos;
  a.n = tokens;
  a.rows = rows;
  a.dim = dim;
  a.chunk = l.chunk;
  a.chunks = l.chunks;
  a.slices = l.slices;
  a.scale = scale;
  a.chunk_base = u32(l.chunk_base);
  a.tile_heads = u32(l.tile_heads);
  a.cap = cap;
  a.out_ids = out_ids;
  a.count = count;
  a.partial = reinterpret_cast<float*>(base + l.partial);
  a.long_list = u32(l.long_list);
  a.long_count = u32(l.long_count);
  using bf = __nv_bfloat16;
  const bool gb = grad_dtype == MUON_BF16, ob = out_dtype == MUON_BF16;
  if (gb && ob) return run_sum<bf, bf>(grad, out, a, stream);
  if (gb) return run_sum<bf, float>(grad, out, a, stream);
  if (ob) return run_sum<float, bf>(grad, out, a, stream);
  return run_sum<float, float>(grad, out, a, stream);
}

}  // namespace muon
