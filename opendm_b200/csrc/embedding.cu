// Token embedding with scaling, and its gradient by sorted tokens.
//
//   lookup    out[t] = round(scale * W[ids[t]])
//   gradient  dW[v]  = round(scale * sum_{t: ids[t] = v} dY[t])
//
// Lookup: a gather bound by HBM (rows in, rows out) for a batch, by latency for a
// few tokens.
//
// Gradient. The tokens are sorted by id (stable, so a row's tokens keep their
// order), then summed:
//   1. sort. Ids left out (padding, out of range) get the key `rows`, which
//      sorts last and is dropped. Up to 2048 tokens in one block, up to
//      32768 in a cluster of eight, more by tiles over the GPU.
//   2. sum. The sorted tokens are cut into chunks of C positions; a warp takes
//      one chunk and 256 columns and adds the rows of dY in sorted order in
//      fp32 registers, writing a row of dW where the key changes. A run of
//      equal keys that goes past its chunk is finished by the warp it starts
//      in, unless it covers the whole next chunk (a "long" run): then each
//      chunk writes its fp32 partial row and the run is put on a list.
//   3. join. Each long run's partial rows are added in chunk order.
// Every sum's order depends on the sorted tokens alone: no floating-point
// atomics, two calls give the same bits.

#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

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

// kE consecutive elements (aligned to all of them, up to 16 bytes) as fp32.
template <int kE, typename T>
__device__ __forceinline__ void load_group(const T* p, float (&v)[kE]) {
  constexpr int kBytes = kE * sizeof(T);
  if constexpr (kBytes > 16) {
    float lo[kE / 2], hi[kE / 2];
    load_group<kE / 2>(p, lo);
    load_group<kE / 2>(p + kE / 2, hi);
#pragma unroll
    for (int i = 0; i < kE / 2; ++i) v[i] = lo[i], v[kE / 2 + i] = hi[i];
  } else if constexpr (kE == 1) {
    if constexpr (sizeof(T) == 2)
      v[0] = __bfloat162float(*p);
    else
      v[0] = *p;
  } else {
    uint32_t w[kBytes / 4];
    if constexpr (kBytes == 16) {
      const uint4 x = *reinterpret_cast<const uint4*>(p);
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else if constexpr (kBytes == 8) {
      const uint2 x = *reinterpret_cast<const uint2*>(p);
      w[0] = x.x, w[1] = x.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
#pragma unroll
    for (int i = 0; i < kBytes / 4; ++i) {
      if constexpr (sizeof(T) == 2) {  // bf16 is the upper half of an fp32
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        v[i] = __uint_as_float(w[i]);
      }
    }
  }
}

template <int kE, typename T>
__device__ __forceinline__ void store_group(T* p, const float (&v)[kE]) {
  constexpr int kBytes = kE * sizeof(T);
  if constexpr (kBytes > 16) {
    float lo[kE / 2], hi[kE / 2];
#pragma unroll
    for (int i = 0; i < kE / 2; ++i) lo[i] = v[i], hi[i] = v[kE / 2 + i];
    store_group<kE / 2>(p, lo);
    store_group<kE / 2>(p + kE / 2, hi);
  } else if constexpr (kE == 1) {
    if constexpr (sizeof(T) == 2)
      *p = __float2bfloat16_rn(v[0]);
    else
      *p = v[0];
  } else {
    uint32_t w[kBytes / 4];
#pragma unroll
    for (int i = 0; i < kBytes / 4; ++i) {
      if constexpr (sizeof(T) == 2) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        w[i] = __float_as_uint(v[i]);
      }
    }
    if constexpr (kBytes == 16)
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (kBytes == 8)
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

// Widest group (8, 4, 2 or 1 elements) that rows of `dim` elements `pitch`
// apart can be cut into, both tensors aligned to it (to 16 bytes at most).
int group_width(int64_t dim, int64_t pitch, const void* a, int a_size, const void* b, int b_size) {
  for (int e = 8; e > 1; e /= 2) {
    const uintptr_t a_bytes = e * a_size < 16 ? e * a_size : 16, b_bytes = e * b_size < 16 ? e * b_size : 16;
    if (dim % e == 0 && pitch % e == 0 && reinterpret_cast<uintptr_t>(a) % a_bytes == 0 &&
        reinterpret_cast<uintptr_t>(b) % b_bytes == 0)
      return e;
  }
  return 1;
}

// ------------------------------------------------------------------ lookup
constexpr int LK_THREADS = 256;
constexpr int LK_PER = 4;

// Rows of whole 8-element groups (16-byte aligned): a block takes 1024
// groups in output order.
template <typename W, typename O>
__global__ void __launch_bounds__(LK_THREADS) lookup_kernel(const W* __restrict__ weight, int64_t rows, int64_t ld,
                                                            const void* __restrict__ ids, bool wide, int64_t tokens,
                                                            uint32_t groups, float scale, O* __restrict__ out,
                                                            int* err) {
  constexpr int kWords = sizeof(W) / 2;  // 16-byte words of a group
  const int64_t base = int64_t(blockIdx.x) * (LK_THREADS * LK_PER);
  const int64_t row0 = base / groups;
  const uint32_t col0 = uint32_t(base - row0 * groups);
  const int64_t left = tokens * groups - base;
  uint4 raw[LK_PER][kWords];
#pragma unroll
  for (int i = 0; i < LK_PER; ++i) {
    const uint32_t o = i * LK_THREADS + threadIdx.x, c = col0 + o, over = c / groups;
    if (o >= left) continue;
    const uint32_t group = c - over * groups;
    const int64_t id = load_id(ids, wide, row0 + over);
    if (id < 0 || id >= rows) {
#pragma unroll
      for (int q = 0; q < kWords; ++q) raw[i][q] = make_uint4(0, 0, 0, 0);
      if (group == 0) record_error(err, MUON_DEV_BAD_INDEX);
    } else {
      const uint4* src = reinterpret_cast<const uint4*>(weight + id * ld) + int64_t(group) * kWords;
#pragma unroll
      for (int q = 0; q < kWords; ++q) raw[i][q] = src[q];
    }
  }
#pragma unroll
  for (int i = 0; i < LK_PER; ++i) {
    const uint32_t o = i * LK_THREADS + threadIdx.x;
    if (o >= left) continue;
    float v[kVec];
    load_group<kVec>(reinterpret_cast<const W*>(raw[i]), v);
#pragma unroll
    for (int k = 0; k < kVec; ++k) v[k] *= scale;
    store_group<kVec>(out + (base + o) * kVec, v);
  }
}

// Other rows: a warp takes up to 1024 columns of one token, eight elements a
// lane at a time in groups of kE (4, 2 or 1): no division per element. The
// fp32 32003 x 1001 table with 40961 tokens into bf16 takes 31.5 us on the
// device and 33.5 a call, against 18.7 of its bytes: loads of 4 and stores of 2
// bytes a lane, so the lines of 164 MB of rows and 82 MB of results cross L2 in
// part sectors. The result is one contiguous array; aligned 16-byte groups over
// two tokens, with the rows read through shared memory, were not tried.
constexpr int LK_COLS = 1024;

// kAnyScale: the scale may be infinite or NaN, which a bad id's zeros must not
// be multiplied by. Looking for that in every call cost up to 11% (20000 x 2052
// bf16 27.7 -> 31.0 us, 2048 fp32 into bf16 28.8 -> 30.7), so such a scale has a
// kernel of its own.
template <int kE, bool kAnyScale, typename W, typename O>
__global__ void __launch_bounds__(LK_THREADS) lookup_rows_kernel(const W* __restrict__ weight, int64_t rows,
                                                                 int64_t ld, const void* __restrict__ ids, bool wide,
                                                                 int64_t tokens, int64_t dim, int64_t parts,
                                                                 float scale, O* __restrict__ out, int* err) {
  constexpr int kGroups = kVec / kE, kStep = 32 * kE;
  const int lane = threadIdx.x & 31;
  const int64_t unit = int64_t(blockIdx.x) * (LK_THREADS / 32) + (threadIdx.x >> 5);
  const int64_t t = unit / parts, part = unit - t * parts;
  if (t >= tokens) return;
  const int64_t id = load_id(ids, wide, t);
  const bool ok = id >= 0 && id < rows;
  const float by = kAnyScale && !ok ? 0.f : scale;
  if (!ok && part == 0 && lane == 0) record_error(err, MUON_DEV_BAD_INDEX);
  const int64_t c0 = part * LK_COLS;
  const int n = static_cast<int>(min(int64_t(LK_COLS), dim - c0)) - lane * kE;  // columns from this lane's first on
  const W* src = weight + (ok ? id * ld : 0) + c0 + lane * kE;
  O* dst = out + t * dim + c0 + lane * kE;
  for (int at = 0; at < n; at += kGroups * kStep) {
    float v[kGroups][kE];
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
#pragma unroll
      for (int i = 0; i < kE; ++i) v[k][i] = 0.f;
      if (ok && at + k * kStep < n) load_group<kE>(src + at + k * kStep, v[k]);
    }
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
#pragma unroll
      for (int i = 0; i < kE; ++i) v[k][i] *= by;
      if (at + k * kStep < n) store_group<kE>(dst + at + k * kStep, v[k]);
    }
  }
}

template <typename W, typename O>
int run_lookup(const void* weight, int64_t rows, int64_t dim, int64_t ld, const void* ids, bool wide, int64_t tokens,
               float scale, void* out, int* err, cudaStream_t stream) {
  const int width = group_width(dim, ld, weight, sizeof(W), out, sizeof(O));
  const bool finite = std::isfinite(scale), flat = finite && width == kVec;
  const int64_t groups = dim / kVec, parts = (dim + LK_COLS - 1) / LK_COLS;
  const int64_t units = flat ? tokens * groups : tokens * parts, per = flat ? LK_THREADS * LK_PER : LK_THREADS / 32;
  const int64_t blocks = (units + per - 1) / per;
  if (blocks > 0x7fffffffLL) return set_error(MUON_ERR_ARG, "embedding output too large");
  const unsigned grid = static_cast<unsigned>(blocks);
  const W* w = static_cast<const W*>(weight);
  O* o = static_cast<O*>(out);
  auto by_rows = [&](auto kernel) {
    kernel<<<grid, LK_THREADS, 0, stream>>>(w, rows, ld, ids, wide, tokens, dim, parts, scale, o, err);
  };
  if (flat)
    lookup_kernel<W, O><<<grid, LK_THREADS, 0, stream>>>(w, rows, ld, ids, wide, tokens,
                                                         static_cast<uint32_t>(groups), scale, o, err);
  else if (!finite)
    by_rows(lookup_rows_kernel<1, true, W, O>);
  else if (width == 4)
    by_rows(lookup_rows_kernel<4, false, W, O>);
  else if (width == 2)
    by_rows(lookup_rows_kernel<2, false, W, O>);
  else
    by_rows(lookup_rows_kernel<1, false, W, O>);
  return check_cuda(cudaGetLastError(), "embedding launch");
}

// -------------------------------------------------------------------- sort
// Least-significant-digit radix sort of (key, position), digits of at most 9
// bits: two passes for vocabularies below 2^18. A warp ranks its keys 32 at a
// time: equal digits find each other with a ballot per bit (16384 tokens in one
// block took 44 us so, and 49 us with match_any), so the order of equal keys
// is kept.
constexpr int RS_BITS = 9;
constexpr int RS_BINS = 1 << RS_BITS;
constexpr int RS_THREADS = RS_BINS;  // a thread a bin
constexpr int RS_WARPS = RS_THREADS / 32;
constexpr int RS_MAX_PASSES = 4;

struct TokenSource {
  const void* ids;
  bool wide;
  int64_t rows;
  int64_t padding;
};

// Key of token t: its id, or `rows` when it takes no part.
__device__ __forceinline__ uint32_t token_key(const TokenSource& s, int64_t t, int* err) {
  const int64_t id = load_id(s.ids, s.wide, t);
  if (id < 0 || id >= s.rows) {
    if (err) record_error(err, MUON_DEV_BAD_INDEX);
    return static_cast<uint32_t>(s.rows);
  }
  return id == s.padding ? static_cast<uint32_t>(s.rows) : static_cast<uint32_t>(id);
}

// Most of the GPU idles while a block or a cluster sorts. In the dense form,
// extra blocks of that kernel write zeros over the last rows of the result; the
// sum writes those of them that have tokens and leaves the rest. 48 MB by 64
// blocks beside a cluster, 8 MB beside one block, against none (us a call):
//   151936 x 2048 bf16  512 tokens 95.4 / 96.4, 2049 101.9 / 102.7, 4096 105.5 /
//     107.3, 8192 109.1 / 111.3, 16384 117.4 / 123.2, 32768 140.1 / 143.9
//   32003 x 1024 fp32   2049 37.9 / 39.8, 16384 51.7 / 58.1, 32768 73.2 / 78.4
//   151936 x 256 bf16   2049 29.6 / 29.7, 8192 31.7 / 32.9, 32768 46.0 / 50.2
// A result little larger than the 48 MB gains at 16384 tokens (50000 x 512 bf16
// 33.3 / 35.8) and loses about 1 us from 3000 to 8192 (30.7 / 29.5); one of 25 MB
// (12000 x 1024 bf16) is between 2 us faster (3000, 8192) and 2 us slower (32768).
// By 32 blocks 16384 tokens of the first took 126 us, by 128 118 (they slow the
// sort), with 64 or 80 MB 117-119. The rows past the count of the row form gained
// nothing so.
struct Fill {
  char* from;  // 16-byte aligned
  int64_t vectors;
  int blocks;
};

__device__ __forceinline__ void fill_zeros(const Fill& f, int block) {
  uint4* v = reinterpret_cast<uint4*>(f.from);
  for (int64_t i = int64_t(block) * blockDim.x + threadIdx.x; i < f.vectors; i += int64_t(f.blocks) * blockDim.x)
    v[i] = make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ uint32_t warp_inclusive(uint32_t x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, x, off);
    if (lane >= off) x += up;
  }
  return x;
}

// Exclusive prefix over a block of RS_THREADS threads; `sums` holds RS_WARPS words.
__device__ __forceinline__ uint32_t block_exclusive(uint32_t x, uint32_t* sums, uint32_t* total = nullptr) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t inc = warp_inclusive(x);
  if (lane == 31) sums[warp] = inc;
  __syncthreads();
  const uint32_t mine = lane < RS_WARPS ? sums[lane] : 0;
  const uint32_t all = warp_inclusive(mine);
  const uint32_t before = __shfl_sync(0xffffffffu, all - mine, warp);
  if (total) *total = __shfl_sync(0xffffffffu, all, 31);
  __syncthreads();
  return before + inc - x;
}

// Lanes whose `d` (of RS_BITS bits) equals this lane's.
__device__ __forceinline__ uint32_t equal_digits(uint32_t d) {
  uint32_t peers = 0xffffffffu;
#pragma unroll
  for (int b = 0; b < RS_BITS; ++b) {
    const bool set = (d >> b) & 1u;
    const uint32_t votes = __ballot_sync(0xffffffffu, set);
    peers &= set ? votes : ~votes;
  }
  return peers;
}

// Stable ranks of a warp's kPer x 32 digits within the warp; counts[digit] ends as the warp's count.
template <int kPer, typename Get>
__device__ __forceinline__ void warp_ranks(uint16_t* counts, uint32_t (&rank)[kPer], Get&& digit) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t d = digit(i);
    const uint32_t peers = equal_digits(d);
    const uint32_t before = __popc(peers & ((1u << lane) - 1u));
    const uint32_t count = counts[d];
    __syncwarp();
    if (before == 0) counts[d] = static_cast<uint16_t>(count + __popc(peers));
    __syncwarp();
    rank[i] = count + before;
  }
}

// counts[warp][bin] -> how many keys of that bin the warps before hold; returns the total of the thread's bin.
__device__ __forceinline__ uint32_t scan_warps(uint16_t (*counts)[RS_BINS]) {
  uint32_t run = 0;
  uint16_t c[RS_WARPS];
#pragma unroll
  for (int w = 0; w < RS_WARPS; ++w) c[w] = counts[w][threadIdx.x];
#pragma unroll
  for (int w = 0; w < RS_WARPS; ++w) {
    counts[w][threadIdx.x] = static_cast<uint16_t>(run);
    run += c[w];
  }
  return run;
}

// counts: aligned to a word, which its element type alone does not ask for
__device__ __forceinline__ void clear_counts(uint16_t (*counts)[RS_BINS]) {
  uint32_t* words = reinterpret_cast<uint32_t*>(counts);
#pragma unroll
  for (int i = 0; i < RS_WARPS * RS_BINS / 2 / RS_THREADS; ++i) words[i * RS_THREADS + threadIdx.x] = 0;
}

constexpr int HD_TILE = 4096;  // positions that share one entry of tile_base

// Run starts among a block's sorted keys (element e0 + 32 i of the warp), as
// ballots; `prev` gives the key before a position.
template <int kPer, typename Prev>
__device__ __forceinline__ uint32_t run_heads(const uint32_t (&key)[kPer], uint32_t rows, uint32_t (&heads)[kPer],
                                              Prev&& prev) {
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t before = prev(i);
    heads[i] = __ballot_sync(0xffffffffu, key[i] != before && key[i] < rows);
    mine += __popc(heads[i]);
  }
  return mine;
}

// Sort of up to RS_THREADS x kPer tokens in one block, with the run starts
// counted on the way out.
template <int kPer>
__global__ void __launch_bounds__(RS_THREADS) block_sort_kernel(TokenSource src, int n, int passes, int bits,
                                                                int chunk, uint32_t* __restrict__ out_keys,
                                                                uint32_t* __restrict__ out_pos,
                                                                uint32_t* __restrict__ chunk_base,
                                                                uint32_t* __restrict__ tile_base,
                                                                uint32_t* __restrict__ long_count,
                                                                int64_t* __restrict__ row_count, int* err, Fill fill) {
  __shared__ uint32_t skey[RS_THREADS * kPer];
  __shared__ __align__(16) uint16_t spos[RS_THREADS * kPer];
  __shared__ __align__(16) uint16_t counts[RS_WARPS][RS_BINS];
  __shared__ __align__(16) uint16_t base[RS_BINS];
  __shared__ uint32_t sums[RS_WARPS];
  allow_next();
  if (blockIdx.x > 0) {
    fill_zeros(fill, blockIdx.x - 1);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int e0 = warp * 32 * kPer + lane;
  const uint32_t rows = static_cast<uint32_t>(src.rows), mask = (1u << bits) - 1u;
  uint32_t key[kPer], pos[kPer];  // element e0 + 32 i; places past n sort last: all digits highest
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    pos[i] = e0 + 32 * i;
    key[i] = e0 + 32 * i < n ? token_key(src, e0 + 32 * i, err) : 0xffffffffu;
  }
  for (int p = 0; p < passes; ++p) {
    const int shift = p * bits;
    clear_counts(counts);
    __syncthreads();
    uint32_t rank[kPer];
    warp_ranks<kPer>(counts[warp], rank, [&](int i) { return (key[i] >> shift) & mask; });
    __syncthreads();
    const uint32_t first = block_exclusive(scan_warps(counts), sums);
    base[threadIdx.x] = static_cast<uint16_t>(first);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t d = (key[i] >> shift) & mask;
      const uint32_t to = base[d] + counts[warp][d] + rank[i];
      skey[to] = key[i];
      spos[to] = static_cast<uint16_t>(pos[i]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      key[i] = skey[e0 + 32 * i];
      pos[i] = spos[e0 + 32 * i];
    }
  }
  uint32_t heads[kPer], total;
  const uint32_t mine = run_heads<kPer>(key, rows, heads, [&](int i) {
    const int e = e0 + 32 * i;
    return e > 0 ? skey[e - 1] : 0xffffffffu;
  });
  uint32_t before = block_exclusive(lane == 0 ? mine : 0, sums, &total);
  before = __shfl_sync(0xffffffffu, before, 0);  // run starts before this warp's first position
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = e0 + 32 * i;
    if (e < n) {
      out_keys[e] = key[i];
      out_pos[e] = pos[i];
      if (e % chunk == 0) chunk_base[e / chunk] = before + __popc(heads[i] & ((1u << lane) - 1u));
    }
    before += __popc(heads[i]);
  }
  if (threadIdx.x == 0) {
    tile_base[0] = 0;
    *long_count = 0;
    if (row_count) *row_count = total;
  }
}

// The same by a cluster of eight blocks for up to 8 x RS_THREADS x kPer
// tokens (one block alone needs 44 us for 16384, bound by its instruction
// issue): digit totals and the scattered keys cross the blocks through
// distributed shared memory. tile_base gets each block's own run starts.
constexpr int CL_BLOCKS = 8;

template <int kPer>
struct ClusterSortShared {
  uint2 recv[RS_THREADS * kPer];  // (key, position) that this block holds after a pass
  __align__(16) uint16_t counts[RS_WARPS][RS_BINS];
  uint32_t totals[RS_BINS];
  uint32_t base[RS_BINS];
  uint32_t sums[RS_WARPS];
};

template <int kPer>
__global__ void __cluster_dims__(CL_BLOCKS, 1, 1) __launch_bounds__(RS_THREADS)
    cluster_sort_kernel(TokenSource src, int n, int passes, int bits, int chunk, uint32_t* __restrict__ out_keys,
                        uint32_t* __restrict__ out_pos, uint32_t* __restrict__ chunk_base,
                        uint32_t* __restrict__ tile_base, uint32_t* __restrict__ long_count, int* err, Fill fill) {
  extern __shared__ __align__(16) unsigned char raw[];
  ClusterSortShared<kPer>& sh = *reinterpret_cast<ClusterSortShared<kPer>*>(raw);
  constexpr int kHeld = RS_THREADS * kPer;
  allow_next();
  if (blockIdx.x >= CL_BLOCKS) {  // whole clusters of their own
    fill_zeros(fill, blockIdx.x - CL_BLOCKS);
    return;
  }
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const unsigned block = cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h0 = warp * 32 * kPer + lane, e0 = int(block) * kHeld + h0;
  const uint32_t rows = static_cast<uint32_t>(src.rows), mask = (1u << bits) - 1u;
  uint32_t key[kPer], pos[kPer];  // element e0 + 32 i; places past n sort last: all digits highest
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = e0 + 32 * i;
    key[i] = e < n ? token_key(src, e, err) : 0xffffffffu;
    pos[i] = e;
  }
  for (int p = 0; p < passes; ++p) {
    const int shift = p * bits;
    clear_counts(sh.counts);
    __syncthreads();
    uint32_t rank[kPer];
    warp_ranks<kPer>(sh.counts[warp], rank, [&](int i) { return (key[i] >> shift) & mask; });
    __syncthreads();
    sh.totals[threadIdx.x] = scan_warps(sh.counts);
    cluster.sync();  // totals written, and recv of the pass before read
    uint32_t all = 0, before = 0;
#pragma unroll
    for (unsigned q = 0; q < CL_BLOCKS; ++q) {
      const uint32_t c = *cluster.map_shared_rank(&sh.totals[threadIdx.x], q);
      all += c;
      if (q < block) before += c;
    }
    const uint32_t first = block_exclusive(all, sh.sums);
    sh.base[threadIdx.x] = first + before;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t d = (key[i] >> shift) & mask;
      const uint32_t to = sh.base[d] + sh.counts[warp][d] + rank[i];
      *cluster.map_shared_rank(&sh.recv[to % kHeld], to / kHeld) = make_uint2(key[i], pos[i]);
    }
    cluster.sync();  // recv written, and totals read
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint2 x = sh.recv[h0 + 32 * i];
      key[i] = x.x;
      pos[i] = x.y;
    }
  }
  uint32_t heads[kPer], total;
  const uint32_t mine = run_heads<kPer>(key, rows, heads, [&](int i) {
    const int h = h0 + 32 * i;
    if (h > 0) return sh.recv[h - 1].x;
    return block > 0 ? cluster.map_shared_rank(&sh.recv[kHeld - 1], block - 1)->x : 0xffffffffu;
  });
  uint32_t before = block_exclusive(lane == 0 ? mine : 0, sh.sums, &total);
  before = __shfl_sync(0xffffffffu, before, 0);  // run starts in this block before this warp's first position
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = e0 + 32 * i;
    if (e < n) {
      out_keys[e] = key[i];
      out_pos[e] = pos[i];
      if (e % chunk == 0) chunk_base[e / chunk] = before + __popc(heads[i] & ((1u << lane) - 1u));
    }
    before += __popc(heads[i]);
  }
  if (threadIdx.x == 0) {
    tile_base[block] = total;
    if (block == 0) *long_count = 0;
  }
  cluster.sync();  // no block leaves while another reads its shared memory
}

// Larger sorts: digit counts of every tile for the first pass, then one
// scatter a pass. A scatter block adds the tiles' counts itself (its first
// positions are the sums over the smaller digits and the tiles before it)
// and counts the next pass's digits by destination tile as it writes. Reading
// all tiles' counts in every block is quadratic, 2 KB x tiles^2 a pass, and next
// to nothing at the sizes of a training batch: a whole call of two fp32 columns
// takes 69 us at 131072 tokens, 126 at 400000, 300 at a million, 1420 at four
// million and 8010 at sixteen. Far above that it rules (a pass over 2^31 tokens
// would read 560 TB): split such a list.
constexpr int RS_PER = 8;
constexpr int RS_TILE = RS_THREADS * RS_PER;

__global__ void __launch_bounds__(RS_THREADS) radix_count_kernel(TokenSource src, int64_t n, int bits, int passes,
                                                                 int64_t tiles, uint32_t* __restrict__ hist,
                                                                 uint32_t* __restrict__ zeroed, int* err) {
  __shared__ uint32_t h[RS_BINS];
  allow_next();
  const int lane = threadIdx.x & 31;
  h[threadIdx.x] = 0;
  for (int p = 1; p < passes; ++p) hist[(p * tiles + blockIdx.x) * RS_BINS + threadIdx.x] = 0;
  if (blockIdx.x == 0 && threadIdx.x < 2) zeroed[threadIdx.x] = 0;
  __syncthreads();
  const int64_t base = int64_t(blockIdx.x) * RS_TILE;
#pragma unroll
  for (int i = 0; i < RS_PER; ++i) {
    const int64_t t = base + i * RS_THREADS + threadIdx.x;
    const uint32_t d = t < n ? token_key(src, t, err) & ((1u << bits) - 1u) : 0;
    const uint32_t peers = equal_digits(d) & __ballot_sync(0xffffffffu, t < n);
    if (t < n && lane == __ffs(peers) - 1)  // one add for the warp's equal digits
      atomicAdd(&h[d], static_cast<uint32_t>(__popc(peers)));
  }
  __syncthreads();
  hist[int64_t(blockIdx.x) * RS_BINS + threadIdx.x] = h[threadIdx.x];
}

__global__ void __launch_bounds__(RS_THREADS) radix_scatter_kernel(TokenSource src, const uint32_t* keys,
                                                                   const uint32_t* positions, int64_t n, int shift,
                                                                   int bits, int64_t tiles, const uint32_t* hist,
                                                                   uint32_t* next_hist, uint32_t* out_keys,
                                                                   uint32_t* out_pos) {
  __shared__ __align__(16) uint16_t counts[RS_WARPS][RS_BINS];
  __shared__ uint32_t base[RS_BINS];
  __shared__ uint32_t sums[RS_WARPS];
  allow_next();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  clear_counts(counts);
  wait_previous();
  // this tile's first position of every digit, a thread a digit (before the keys are asked for: behind them a call
  // of 400000 tokens x 2 took 139 us, not 126)
  uint32_t before = 0, total = 0;
#pragma unroll 16
  for (int64_t t = 0; t < tiles; ++t) {
    const uint32_t c = hist[t * RS_BINS + threadIdx.x];
    total += c;
    if (t < int64_t(blockIdx.x)) before += c;
  }
  const int64_t e0 = int64_t(blockIdx.x) * RS_TILE + warp * 32 * RS_PER + lane;
  const uint32_t mask = (1u << bits) - 1u;
  uint32_t key[RS_PER], pos[RS_PER], rank[RS_PER];
#pragma unroll
  for (int i = 0; i < RS_PER; ++i) {
    const int64_t e = e0 + 32 * i;
    key[i] = 0xffffffffu;
    pos[i] = static_cast<uint32_t>(e);
    if (e < n) {
      key[i] = keys ? keys[e] : token_key(src, e, nullptr);
      if (keys) pos[i] = positions[e];
    }
  }
  __syncthreads();
  warp_ranks<RS_PER>(counts[warp], rank, [&](int i) { return (key[i] >> shift) & mask; });
  const uint32_t first = block_exclusive(total, sums);
  base[threadIdx.x] = first + before;
  scan_warps(counts);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RS_PER; ++i) {
    const bool in = e0 + 32 * i < n;
    const uint32_t d = (key[i] >> shift) & mask;
    const uint32_t to = base[d] + counts[warp][d] + rank[i];
    if (in) {
      out_keys[to] = key[i];
      out_pos[to] = pos[i];
    }
    if (next_hist) {  // one add for the lanes whose next digit and tile are those of the first lane of that digit
      const uint32_t d2 = (key[i] >> (shift + bits)) & mask, tile = to / RS_TILE;
      const uint32_t peers = equal_digits(d2) & __ballot_sync(0xffffffffu, in);
      const int leader = in ? __ffs(peers) - 1 : lane;
      const bool same = __shfl_sync(0xffffffffu, tile, leader) == tile;
      const uint32_t joined = peers & __ballot_sync(0xffffffffu, in && same);
      if (in && (lane == leader || !same))
        atomicAdd(&next_hist[tile * RS_BINS + d2], lane == leader ? static_cast<uint32_t>(__popc(joined)) : 1u);
    }
  }
}

// How many runs start before each chunk: chunk_base[c] within the chunk's
// tile of HD_TILE positions, tile_base[t] before the tile (by the last block to
// finish), and their number.
constexpr int HD_THREADS = 1024;

__global__ void __launch_bounds__(HD_THREADS) heads_kernel(const uint32_t* keys, int64_t n, uint32_t rows, int chunk,
                                                           uint32_t* chunk_base, uint32_t* tile_base, uint32_t* ticket,
                                                           int64_t* row_count) {
  constexpr int kWarps = HD_THREADS / 32, kRounds = HD_TILE / HD_THREADS;
  __shared__ uint32_t warp_sum[kWarps];
  __shared__ uint32_t last;
  allow_next();
  wait_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t e0 = int64_t(blockIdx.x) * HD_TILE + warp * 32 * kRounds + lane;
  uint32_t heads[kRounds], key[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) key[i] = e0 + 32 * i < n ? keys[e0 + 32 * i] : 0xffffffffu;
  const uint32_t edge = lane == 0 && e0 > 0 && e0 <= n ? keys[e0 - 1] : 0xffffffffu;  // before the warp's first
  const uint32_t mine = run_heads<kRounds>(key, rows, heads, [&](int i) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, key[i], 1);
    const uint32_t wrap = i > 0 ? __shfl_sync(0xffffffffu, key[i > 0 ? i - 1 : 0], 31) : edge;
    return lane > 0 ? up : wrap;
  });
  if (lane == 0) warp_sum[warp] = mine;
  __syncthreads();
  uint32_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int64_t e = e0 + 32 * i;
    if (e < n && e % chunk == 0) chunk_base[e / chunk] = before + __popc(heads[i] & ((1u << lane) - 1u));
    before += __popc(heads[i]);
  }
  if (threadIdx.x == 0) {
    tile_base[blockIdx.x] = total;
    __threadfence();
    last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  uint32_t run = 0;
  for (unsigned t0 = 0; t0 < gridDim.x; t0 += HD_THREADS) {
    const unsigned t = t0 + threadIdx.x;
    const uint32_t x = t < gridDim.x ? *reinterpret_cast<volatile uint32_t*>(tile_base + t) : 0;
    const uint32_t inc = warp_inclusive(x);
    __syncthreads();
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    uint32_t pre = run + inc - x;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) pre += warp_sum[w];
      run += warp_sum[w];
    }
    if (t < gridDim.x) tile_base[t] = pre;
  }
  if (threadIdx.x == 0 && row_count) *row_count = run;
}

// --------------------------------------------------------------------- sum
constexpr int SUM_THREADS = 256;
constexpr int SUM_WARPS = SUM_THREADS / 32;
constexpr int SUM_STAGE_BYTES = 4096;  // rows in flight of one warp
constexpr int64_t ZERO_BYTES = 8192;   // of rows one warp of the zero part looks after

// A lane's 8 of a slice's 256 columns: groups of kE, 32 kE columns apart.
template <int kE, typename T>
__device__ __forceinline__ void store_cols(T* row, int64_t slice, int64_t dim, const float (&v)[kVec]) {
  const int64_t col = slice * kSlice + (threadIdx.x & 31) * kE;
#pragma unroll
  for (int k = 0; k < kVec / kE; ++k) {
    float g[kE];
#pragma unroll
    for (int i = 0; i < kE; ++i) g[i] = v[k * kE + i];
    if (col + k * 32 * kE < dim) store_group<kE>(row + col + k * 32 * kE, g);
  }
}

struct LongRun {
  uint32_t chunk;  // the chunk it starts in
  uint32_t parts;  // how many chunks it reaches
  int64_t row;     // of the result
};

struct SumArgs {
  const uint32_t* keys;
  const uint32_t* pos;
  int64_t n;
  int64_t rows;
  int64_t dim;
  int chunk;
  int64_t chunks;
  int64_t slices;
  int64_t sum_blocks;
  int64_t zero_rows;  // rows of a warp that writes zeros
  int64_t filled;     // dense form: the rows from here on were filled with zeros before
  float scale;
  const uint32_t* chunk_base;
  const uint32_t* tile_base;
  int64_t tile;    // positions that share one entry of tile_base
  int raw_tiles;   // entries of tile_base that hold counts of their own, to be added up (0: sums already)
  int64_t cap;
  int64_t* out_ids;  // NULL: dense form
  int64_t* count;
  float* partial;  // [chunks][2][slices * kSlice]: a run from an earlier chunk; a long run starting here
  LongRun* long_list;
  uint32_t* long_count;
};

// Run starts before tile `t` (t = raw_tiles: all of them), by a whole warp.
__device__ __forceinline__ uint32_t heads_before(const SumArgs& a, int t) {
  if (a.raw_tiles == 0) return a.tile_base[t];
  const int lane = threadIdx.x & 31;
  return __reduce_add_sync(0xffffffffu, lane < t ? a.tile_base[lane] : 0u);
}

// First index in keys[lo, hi) whose key is >= `key`, by a whole warp: 32
// probes a step, four dependent loads for a million tokens.
__device__ __forceinline__ int64_t warp_lower_bound(const uint32_t* keys, int64_t lo, int64_t hi, int64_t key) {
  const int lane = threadIdx.x & 31;
  while (lo < hi) {
    const int64_t step = (hi - lo + 31) / 32;
    const int64_t at = lo + int64_t(lane) * step;
    const bool below = at < hi && int64_t(keys[at]) < key;
    const int k = __popc(__ballot_sync(0xffffffffu, below));  // the probes below `key` come first
    if (k == 0) return lo;
    const int64_t last_below = lo + int64_t(k - 1) * step;
    hi = min(hi, last_below + step);
    lo = last_below + 1;
  }
  return lo;
}

// Zeros elements [begin, end) of out, by a warp.
template <typename O>
__device__ __forceinline__ void zero_span(O* out, int64_t begin, int64_t end) {
  constexpr int kPer = 16 / sizeof(O);
  const int lane = threadIdx.x & 31;
  const float zero[1] = {0.f};
  const int64_t skew = (reinterpret_cast<uintptr_t>(out) / sizeof(O)) % kPer;  // elements past a 16-byte boundary
  const int64_t body = min(end, (begin + skew + kPer - 1) / kPer * kPer - skew);
  for (int64_t e = begin + lane; e < body; e += 32) store_group<1>(out + e, zero);
  const int64_t vectors = (end - body) / kPer;
  uint4* v = reinterpret_cast<uint4*>(out + body);
  for (int64_t i = lane; i < vectors; i += 32) v[i] = make_uint4(0, 0, 0, 0);
  for (int64_t e = body + vectors * kPer + lane; e < end; e += 32) store_group<1>(out + e, zero);
}

// Rows no token has: in the dense form the gaps between the sorted keys, in
// the row form those past the count.
template <typename O>
__device__ __forceinline__ void zero_rows(O* out, const SumArgs& a, int64_t unit) {
  const int lane = threadIdx.x & 31;
  const int64_t r0 = unit * a.zero_rows;
  if (a.out_ids) {
    const int64_t count = a.raw_tiles ? int64_t(heads_before(a, a.raw_tiles)) : *a.count;
    if (a.raw_tiles && unit == 0 && lane == 0) *a.count = count;
    const int64_t from = max(r0, count), to = min(r0 + a.zero_rows, a.cap);
    if (from >= to) return;
    zero_span(out, from * a.dim, to * a.dim);
    if (from + lane < to) a.out_ids[from + lane] = 0;
    return;
  }
  const int n = static_cast<int>(min(a.zero_rows, a.filled - r0));  // at most 32
  if (n <= 0) return;
  // which of the rows have tokens, a bit each: 32 sorted keys at a time, long runs skipped by a search
  uint32_t taken = 0;
  int64_t at = warp_lower_bound(a.keys, 0, a.n, r0);
  while (at < a.n) {
    const uint32_t key = at + lane < a.n ? a.keys[at + lane] : 0xffffffffu;
    const bool mine = int64_t(key) < r0 + n;
    taken |= __reduce_or_sync(0xffffffffu, mine ? 1u << (key - uint32_t(r0)) : 0u);
    if (!__all_sync(0xffffffffu, mine)) break;
    const uint32_t first = __shfl_sync(0xffffffffu, key, 0), last = __shfl_sync(0xffffffffu, key, 31);
    at = first == last ? warp_lower_bound(a.keys, at + 32, a.n, int64_t(last) + 1) : at + 32;
  }
  uint32_t empty = ~taken & (n == 32 ? 0xffffffffu : (1u << n) - 1u);
  while (empty) {  // spans of rows without tokens
    const int from = __ffs(empty) - 1;
    const uint32_t above = ~(empty >> from);
    const int span = above ? __ffs(above) - 1 : 32;
    zero_span(out, (r0 + from) * a.dim, (r0 + from + span) * a.dim);
    if (from + span >= 32) break;
    empty &= ~0u << (from + span);
  }
}

template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t shared, const void* global) {
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared), "l"(global) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(shared), "l"(global), "n"(kBytes) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// One chunk and 256 columns a warp, eight columns a lane in groups of kE. The
// rows of dY come through a ring in shared memory (4 KB a warp, filled by
// asynchronous copies that each lane makes and reads for itself), so few
// registers are held; single bf16 elements, too small for such copies, are
// loaded two rows at a time instead (six blocks an SM: a call of 50000 x 1001 146
// us, with four rows 150, with five blocks 161). 131072 x 2560 bf16 into rows: 184 us,
// 6.6 TB/s of DRAM traffic.
// A small batch is bound by the issue slots and its one wave of blocks: 16384 x
// 2048 24 us; 16 columns a lane cost it 3 us more. The blocks behind sum_blocks
// write the zeros, 8 KB of rows a warp: with 64 KB the dense gradient of 16384
// tokens (151936 x 2048) took 106-124 us, not 99, and zeros laid among the other
// blocks 117.
template <int kE, typename G, typename O>
__global__ void __launch_bounds__(SUM_THREADS, kE * sizeof(G) >= 4 ? 1 : 6)
    sum_kernel(const G* grad, O* out, const SumArgs a) {
  constexpr bool kRing = kE * sizeof(G) >= 4;
  constexpr int kStages = SUM_STAGE_BYTES / (kSlice * int(sizeof(G)));
  constexpr int kGroups = kVec / kE, kGroupBytes = kE * sizeof(G);
  static_assert(kGroupBytes <= 16, "one asynchronous copy a group");
  __shared__ __align__(16) unsigned char ring[kRing ? SUM_WARPS : 1][kRing ? SUM_STAGE_BYTES : 16];
  __shared__ int64_t held_row[SUM_WARPS][2 * kMaxChunk];  // first element of the rows of this chunk and the next
  __shared__ uint32_t held_key[SUM_WARPS][2 * kMaxChunk];
  allow_next();
  wait_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (int64_t(blockIdx.x) >= a.sum_blocks) {
    zero_rows(out, a, (int64_t(blockIdx.x) - a.sum_blocks) * SUM_WARPS + warp);
    return;
  }
  const int64_t unit = int64_t(blockIdx.x) * SUM_WARPS + warp;
  const int64_t c = unit / a.slices;
  if (c >= a.chunks) return;
  const int64_t slice = unit - c * a.slices;
  const int64_t s0 = c * a.chunk;
  const int len = static_cast<int>(min(int64_t(a.chunk), a.n - s0));
  const int64_t s1 = s0 + len;
  const int next = static_cast<int>(min(int64_t(a.chunk), a.n - s1));
  const uint32_t none = 0xffffffffu;
  const uint32_t dropped = static_cast<uint32_t>(a.rows);
  // keys and positions of this chunk and the next, one per lane each
  const uint32_t key_a = lane < len ? a.keys[s0 + lane] : none;
  const uint32_t key_b = lane < next ? a.keys[s1 + lane] : none;
  const uint32_t pos_a = lane < len ? a.pos[s0 + lane] : 0;
  const uint32_t pos_b = lane < next ? a.pos[s1 + lane] : 0;
  const uint32_t before = s0 > 0 ? a.keys[s0 - 1] : none;
  const uint32_t before_last = s0 > a.chunk ? a.keys[s0 - a.chunk - 1] : none;
  uint32_t slot = a.chunk_base[c] + heads_before(a, static_cast<int>(s0 / a.tile));
  const uint32_t first = __shfl_sync(0xffffffffu, key_a, 0);
  const uint32_t last = __shfl_sync(0xffffffffu, key_a, len - 1);
  const uint32_t next_first = __shfl_sync(0xffffffffu, key_b, 0);
  const uint32_t next_last = __shfl_sync(0xffffffffu, key_b, a.chunk - 1);  // `none` unless the next chunk is full
  const int valid = __popc(__ballot_sync(0xffffffffu, key_a < dropped));
  const bool whole = len == a.chunk && first == last;
  int begin = 0;  // first position this warp adds
  int lead = 0;   // positions of a long run of an earlier chunk
  if (s0 > 0 && before == first) {
    const int run = __popc(__ballot_sync(0xffffffffu, key_a == first));
    if (whole || before_last == first)
      lead = run;
    else
      begin = run;  // the warp of the chunk before finishes this run
  }
  // end of the rows this warp adds: the chunk, plus the rest of a run that does not cover the next chunk
  int end = len;
  bool tail = false;  // a long run starts here
  if (begin < len && lead < len && next_first == last) {
    if (next_last == last)
      tail = true;
    else
      end = len + __popc(__ballot_sync(0xffffffffu, key_b == last));
  }
  if (valid < len) end = valid, tail = false;
  if (begin >= end) return;
  // where a sum is to be written: at the end of a run, and of this warp's part of one
  const uint32_t after_a = __shfl_down_sync(0xffffffffu, key_a, 1), after_b = __shfl_down_sync(0xffffffffu, key_b, 1);
  const uint32_t ends_a =
      __ballot_sync(0xffffffffu, lane < len && key_a != (lane == len - 1 ? next_first : after_a));
  const uint32_t ends_b = __ballot_sync(0xffffffffu, lane < next && (lane == next - 1 || key_b != after_b));
  uint64_t ends = (ends_a | uint64_t(ends_b) << len | uint64_t(1) << (end - 1)) >> begin;
  if (lane < len) held_row[warp][lane] = pos_a * a.dim, held_key[warp][lane] = key_a;
  if (lane < next) held_row[warp][len + lane] = pos_b * a.dim, held_key[warp][len + lane] = key_b;
  __syncwarp();
  const int64_t col = slice * kSlice + lane * kE;
  const int64_t pitch = a.slices * kSlice;
  const G* first_col = grad + col;

  float acc[kVec] = {};
  auto write = [&](int r) {  // the sum that ends with row r
    float* part = a.partial + c * 2 * pitch + slice * kSlice + lane * kVec;
    if (r < lead) {
      store_group<kVec>(part, acc);
    } else if (tail && r == end - 1) {
      store_group<kVec>(part + pitch, acc);
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j) acc[j] *= a.scale;
      const uint32_t key = held_key[warp][r];
      const int64_t row = a.out_ids ? int64_t(slot) : int64_t(key);
      store_cols<kE>(out + row * a.dim, slice, a.dim, acc);
      if (a.out_ids && slice == 0 && lane == 0) a.out_ids[slot] = key;
      ++slot;
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j) acc[j] = 0.f;
  };
  if constexpr (kRing) {
    constexpr int kStageBytes = kSlice * int(sizeof(G));
    const unsigned char* mine = ring[warp] + lane * kGroupBytes;
    const uint32_t mine_to = smem_u32(mine);
    auto fetch = [&](int r, int stage) {
      const G* row = first_col + held_row[warp][r];
#pragma unroll
      for (int k = 0; k < kGroups; ++k)
        if (col + k * 32 * kE < a.dim)
          copy_async<kGroupBytes>(mine_to + stage + k * 32 * kGroupBytes, row + k * 32 * kE);
    };
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      if (begin + i < end) fetch(begin + i, i * kStageBytes);
      copy_async_commit();
    }
    int stage = 0;
    for (int r = begin; r < end; ++r) {
      copy_async_wait<kStages - 1>();
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        float v[kE];
        load_group<kE>(reinterpret_cast<const G*>(mine + stage + k * 32 * kGroupBytes), v);
#pragma unroll
        for (int i = 0; i < kE; ++i) acc[k * kE + i] += v[i];
      }
      if (r + kStages < end) fetch(r + kStages, stage);
      copy_async_commit();
      stage = (stage + kStageBytes) % SUM_STAGE_BYTES;
      if (ends & 1u) write(r);
      ends >>= 1;
    }
  } else {
    constexpr int kAhead = 2;
    for (int r0 = begin; r0 < end; r0 += kAhead) {
      float v[kAhead][kVec];
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        if (r0 + q >= end) continue;
        const G* row = first_col + held_row[warp][r0 + q];
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          float x[1] = {0.f};
          if (col + 32 * k < a.dim) load_group<1>(row + 32 * k, x);
          v[q][k] = x[0];
        }
      }
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        if (r0 + q >= end) continue;
#pragma unroll
        for (int k = 0; k < kVec; ++k) acc[k] += v[q][k];
        if (ends & 1u) write(r0 + q);
        ends >>= 1;
      }
    }
  }
  if (tail && slice == 0) {  // list the run for the join: it reaches the last chunk whose first key is its own
    const int64_t stop = (warp_lower_bound(a.keys, s1, a.n, int64_t(last) + 1) - 1) / a.chunk;
    if (lane == 0) {
      a.long_list[atomicAdd(a.long_count, 1u)] = {uint32_t(c), uint32_t(stop - c + 1),
                                                  a.out_ids ? int64_t(slot) : int64_t(last)};
      if (a.out_ids) a.out_ids[slot] = last;
    }
  }
}

// -------------------------------------------------------------------- join
// One block per (long run, slice): the run's partial rows, split evenly over
// the warps in chunk order, then the warps' sums in order.
template <int kE, typename O>
__global__ void __launch_bounds__(SUM_THREADS) join_kernel(O* out, const SumArgs a) {
  __shared__ __align__(16) float red[SUM_WARPS][kSlice];  // stored in vectors
  wait_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t pitch = a.slices * kSlice;
  const int64_t jobs = int64_t(*a.long_count) * a.slices;
  for (int64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
    const LongRun run = a.long_list[job / a.slices];
    const int64_t slice = job % a.slices, n_parts = run.parts;
    const int64_t per = (n_parts + SUM_WARPS - 1) / SUM_WARPS;
    const int64_t p0 = min(n_parts, warp * per), p1 = min(n_parts, p0 + per);
    float acc[kVec] = {};
    const float* part = a.partial + int64_t(run.chunk) * 2 * pitch + slice * kSlice + lane * kVec;
#pragma unroll 8
    for (int64_t p = p0; p < p1; ++p) {
      float v[kVec];
      load_group<kVec>(part + (p * 2 + (p == 0 ? 1 : 0)) * pitch, v);
#pragma unroll
      for (int j = 0; j < kVec; ++j) acc[j] += v[j];
    }
    store_group<kVec>(&red[warp][lane * kVec], acc);
    __syncthreads();
    if (warp == 0) {
      float w[kVec];
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        float sum = 0.f;
        for (int q = 0; q < SUM_WARPS; ++q) sum += red[q][lane * kVec + j];
        w[j] = sum * a.scale;
      }
      store_cols<kE>(out + run.row * a.dim, slice, a.dim, w);
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

// Chunk length: long chunks leave fewer partial rows to join, short ones give
// more warps (counted in whole slices: a warp of a narrow row does little).
// Calls with at least 32 / 16 / 8 positions: 9000 x 250 (bf16) 31.0 / 29.0 / 28.0
// us, 131072 x 64 65 / 69 / 80, 400000 x 2 (fp32) 108 / 126 / 167 (long runs then
// have ever more parts); 16384 x 2048 takes 48 with 32 whichever is the least. So 16
// above 8192 tokens costs narrow rows of many tokens 4 to 17% and gains 6% at 9000.
int chunk_for(int64_t tokens, int64_t dim) {
  const int least = tokens > 8192 ? 16 : 8;
  int chunk = kMaxChunk;
  while (chunk > least && tokens / chunk * dim < 148 * 16 * kSlice) chunk /= 2;
  return chunk;
}

constexpr int64_t FILL_BLOCK = int64_t(8) << 20, FILL_CLUSTER = int64_t(48) << 20;  // bytes beside either sort
constexpr int64_t FILL_LEAST = int64_t(1) << 20;
constexpr int FILL_BLOCKS = 64;  // a multiple of CL_BLOCKS
static_assert(FILL_BLOCKS % CL_BLOCKS == 0, "whole clusters");

constexpr int64_t kClusterSort = CL_BLOCKS * RS_THREADS * 8;  // tokens; more are sorted by tiles

struct GradLayout {
  int64_t keys[2], pos[2], hist, chunk_base, tile_base, long_list, counters, partial, total;
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
  l.chunk = chunk_for(n, dim);
  l.chunks = (n + l.chunk - 1) / l.chunk;
  for (int i = 0; i < 2; ++i) l.keys[i] = take(4 * n), l.pos[i] = take(4 * n);
  l.hist = take(n > kClusterSort ? 4 * RS_MAX_PASSES * l.tiles * RS_BINS : 0);
  l.chunk_base = take(4 * l.chunks);
  l.tile_base = take(4 * ((n + HD_TILE - 1) / HD_TILE + CL_BLOCKS));
  l.long_list = take(sizeof(LongRun) * l.chunks);
  l.counters = take(8);  // long runs, finished blocks of heads_kernel
  l.partial = take(8 * l.chunks * l.slices * kSlice);
  l.total = at;
  return l;
}

bool float_type(int dtype) { return dtype == MUON_BF16 || dtype == MUON_F32; }
unsigned bytes_of(int float_dtype) { return float_dtype == MUON_BF16 ? 2 : 4; }

// elements x 4 bytes must fit an int64 with room to spare
bool too_large(int64_t a, int64_t b) { return b > 0 && a > (int64_t(1) << 58) / b; }

template <int kE, typename G, typename O>
int run_sum(const void* grad, void* out, const SumArgs& a, unsigned grid, cudaStream_t stream) {
  const G* g = static_cast<const G*>(grad);
  O* o = static_cast<O*>(out);
  if (int rc = launch_overlapped("embedding gradient sum launch", sum_kernel<kE, G, O>, grid, SUM_THREADS, stream, g, o,
                                 a))
    return rc;
  const unsigned join_grid = static_cast<unsigned>(std::min<int64_t>(a.chunks * a.slices, 148 * 8));
  return launch_overlapped("embedding gradient join launch", join_kernel<kE, O>, join_grid, SUM_THREADS, stream, o, a);
}

template <typename G, typename O>
int run_sum(const void* grad, void* out, SumArgs a, cudaStream_t stream) {
  a.sum_blocks = (a.chunks * a.slices + SUM_WARPS - 1) / SUM_WARPS;
  const int64_t row_bytes = a.dim * int64_t(sizeof(O)), rows = a.out_ids ? a.cap : a.filled;
  a.zero_rows = std::clamp(ZERO_BYTES / row_bytes, int64_t(1), int64_t(32));  // a lane or a bit each
  const int64_t blocks = a.sum_blocks + (rows + a.zero_rows * SUM_WARPS - 1) / (a.zero_rows * SUM_WARPS);
  if (blocks > 0x7fffffffLL) return set_error(MUON_ERR_ARG, "embedding gradient too large");
  const unsigned grid = static_cast<unsigned>(blocks);
  switch (group_width(a.dim, a.dim, grad, sizeof(G), out, sizeof(O))) {
    case 8:
      if constexpr (sizeof(G) == 2) return run_sum<8, G, O>(grad, out, a, grid, stream);  // else as four
    case 4:
      return run_sum<4, G, O>(grad, out, a, grid, stream);
    case 2:
      return run_sum<2, G, O>(grad, out, a, grid, stream);
    default:
      return run_sum<1, G, O>(grad, out, a, grid, stream);
  }
}

}  // namespace

int launch_embedding(const void* weight, int weight_dtype, int64_t rows, int64_t dim, int64_t ld, const void* ids,
                     int ids_dtype, int64_t tokens, float scale, void* out, int out_dtype, int* err,
                     cudaStream_t stream) {
  if (rows < 0 || dim < 0 || tokens < 0 || ld < dim)
    return set_error(MUON_ERR_ARG, "negative embedding size or ld < dim");
  if (!float_type(weight_dtype) || !float_type(out_dtype))
    return set_error(MUON_ERR_ARG, "embedding dtypes must be MUON_BF16 or MUON_F32");
  if (ids_dtype != MUON_I32 && ids_dtype != MUON_I64)
    return set_error(MUON_ERR_ARG, "ids must be MUON_I32 or MUON_I64");
  if (too_large(rows, ld) || too_large(tokens, dim) || dim >= kMaxIndex)
    return set_error(MUON_ERR_ARG, "embedding too large");
  if (tokens == 0 || dim == 0) return MUON_OK;
  if ((rows > 0 && !weight) || !ids || !out || !err) return set_error(MUON_ERR_ARG, "null embedding pointer");
  if (misaligned(weight, bytes_of(weight_dtype)) || misaligned(ids, ids_dtype == MUON_I64 ? 8 : 4) ||
      misaligned(out, bytes_of(out_dtype)) || misaligned(err, 4))
    return set_error(MUON_ERR_ARG, "embedding pointer not aligned to its dtype");
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
  if (ids_dtype != MUON_I32 && ids_dtype != MUON_I64)
    return set_error(MUON_ERR_ARG, "ids must be MUON_I32 or MUON_I64");
  if (padding_idx != -1 && (padding_idx < 0 || padding_idx >= rows))
    return set_error(MUON_ERR_ARG, "padding_idx must be -1 or a row");
  if (out_ids && !count) return set_error(MUON_ERR_ARG, "the row form needs a count");
  const int64_t cap = tokens < rows ? tokens : rows;
  const int64_t out_rows = out_ids ? cap : rows;
  if (out_rows * dim > 0 && !out) return set_error(MUON_ERR_ARG, "null embedding gradient output");
  if (tokens > 0 && (!ids || !err || (dim > 0 && !grad)))
    return set_error(MUON_ERR_ARG, "null embedding gradient pointer");
  if (misaligned(grad, bytes_of(grad_dtype)) || misaligned(ids, ids_dtype == MUON_I64 ? 8 : 4) ||
      misaligned(out, bytes_of(out_dtype)) || misaligned(out_ids, 8) || misaligned(count, 8) || misaligned(err, 4))
    return set_error(MUON_ERR_ARG, "embedding gradient pointer not aligned to its dtype");
  const int64_t out_bytes = rows * dim * (out_dtype == MUON_BF16 ? 2 : 4);
  if (tokens == 0 || rows == 0 || dim == 0) {
    if (out_ids) {
      if (check_cuda(cudaMemsetAsync(count, 0, sizeof(int64_t), stream), "embedding gradient count"))
        return MUON_ERR_CUDA;
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
  const TokenSource src{ids, ids_dtype == MUON_I64, rows, padding_idx};
  uint32_t* counters = u32(l.counters);
  int64_t* row_count = out_ids ? count : nullptr;
  SumArgs a{};
  a.tile = HD_TILE;
  int cur = 0;
  a.filled = rows;
  if (tokens <= kClusterSort) {
    const int n = static_cast<int>(tokens);
    Fill fill{};
    if (!out_ids) {
      const int64_t row_bytes = dim * (out_dtype == MUON_BF16 ? 2 : 4);
      const int64_t take = std::min((n <= 4 * RS_THREADS ? FILL_BLOCK : FILL_CLUSTER) / row_bytes, rows);
      const uintptr_t from = reinterpret_cast<uintptr_t>(out) + (rows - take) * row_bytes;
      if (from % 16 == 0 && take * row_bytes % 16 == 0 && take * row_bytes >= FILL_LEAST) {
        fill.from = reinterpret_cast<char*>(from);
        fill.vectors = take * row_bytes / 16;
        fill.blocks = FILL_BLOCKS;
        a.filled = rows - take;
      }
    }
    auto cluster_sort = [&](auto kernel, int per_thread, size_t smem) {
      if (smem > 48 * 1024 &&
          check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)),
                     "cluster sort attribute"))
        return int(MUON_ERR_CUDA);
      kernel<<<CL_BLOCKS + fill.blocks, RS_THREADS, smem, stream>>>(src, n, passes, per, l.chunk, u32(l.keys[0]),
                                                                    u32(l.pos[0]), u32(l.chunk_base),
                                                                    u32(l.tile_base), counters, err, fill);
      a.tile = RS_THREADS * per_thread;
      a.raw_tiles = CL_BLOCKS;
      return int(MUON_OK);
    };
    int rc = MUON_OK;
    auto block_sort = [&](auto kernel) {
      kernel<<<1 + fill.blocks, RS_THREADS, 0, stream>>>(src, n, passes, per, l.chunk, u32(l.keys[0]), u32(l.pos[0]),
                                                         u32(l.chunk_base), u32(l.tile_base), counters, row_count,
                                                         err, fill);
    };
    if (n <= RS_THREADS)
      block_sort(block_sort_kernel<1>);
    else if (n <= RS_THREADS * 4)
      block_sort(block_sort_kernel<4>);
    else if (n <= CL_BLOCKS * RS_THREADS * 2)
      rc = cluster_sort(cluster_sort_kernel<2>, 2, sizeof(ClusterSortShared<2>));
    else if (n <= CL_BLOCKS * RS_THREADS * 4)
      rc = cluster_sort(cluster_sort_kernel<4>, 4, sizeof(ClusterSortShared<4>));
    else
      rc = cluster_sort(cluster_sort_kernel<8>, 8, sizeof(ClusterSortShared<8>));
    if (rc != MUON_OK) return rc;
    if (check_cuda(cudaGetLastError(), "token sort launch")) return MUON_ERR_CUDA;
  } else {
    const unsigned tiles = static_cast<unsigned>(l.tiles);
    radix_count_kernel<<<tiles, RS_THREADS, 0, stream>>>(src, tokens, per, passes, l.tiles, u32(l.hist), counters,
                                                         err);
    if (check_cuda(cudaGetLastError(), "radix count launch")) return MUON_ERR_CUDA;
    const uint32_t *keys = nullptr, *pos = nullptr;
    for (int p = 0; p < passes; ++p) {
      cur = p & 1;
      uint32_t* hist = u32(l.hist) + p * l.tiles * RS_BINS;
      if (int rc = launch_overlapped("radix scatter launch", radix_scatter_kernel, tiles, RS_THREADS, stream, src, keys,
                                     pos, tokens, p * per, per, l.tiles, hist,
                                     p + 1 < passes ? hist + l.tiles * RS_BINS : nullptr, u32(l.keys[cur]),
                                     u32(l.pos[cur])))
        return rc;
      keys = u32(l.keys[cur]);
      pos = u32(l.pos[cur]);
    }
    const unsigned grid = static_cast<unsigned>((tokens + HD_TILE - 1) / HD_TILE);
    if (int rc = launch_overlapped("run heads launch", heads_kernel, grid, HD_THREADS, stream, keys, tokens,
                                   static_cast<uint32_t>(rows), l.chunk, u32(l.chunk_base), u32(l.tile_base),
                                   counters + 1, row_count))
      return rc;
  }
  a.keys = u32(l.keys[cur]);
  a.pos = u32(l.pos[cur]);
  a.n = tokens;
  a.rows = rows;
  a.dim = dim;
  a.chunk = l.chunk;
  a.chunks = l.chunks;
  a.slices = l.slices;
  a.scale = scale;
  a.chunk_base = u32(l.chunk_base);
  a.tile_base = u32(l.tile_base);
  a.cap = cap;
  a.out_ids = out_ids;
  a.count = count;
  a.partial = reinterpret_cast<float*>(base + l.partial);
  a.long_list = reinterpret_cast<LongRun*>(base + l.long_list);
  a.long_count = counters;
  using bf = __nv_bfloat16;
  const bool gb = grad_dtype == MUON_BF16, ob = out_dtype == MUON_BF16;
  if (gb && ob) return run_sum<bf, bf>(grad, out, a, stream);
  if (gb) return run_sum<bf, float>(grad, out, a, stream);
  if (ob) return run_sum<float, bf>(grad, out, a, stream);
  return run_sum<float, float>(grad, out, a, stream);
}

}  // namespace muon
