// Norm of a list of gradients, and clipping in place or into other tensors.
//
//   total = (sum |g|^p)^(1/p), p = 1, 2, inf;  coef = min(max_norm / (total + 1e-6), 1)
//   out   = round(g * coef)
//
// Two launches: the norm pass leaves one double per block, the scale pass
// adds those (every block the same sum in the same order) and rescales. HBM
// bound: one read for the norm, one read and one write for the scaling. 239 M
// bf16 elements in 37 tensors: 236 us, 6.1 TB/s of those bytes; 302 M fp32
// into bf16: 461-470 us, 6.4-6.5 TB/s. The scale pass walks the list backwards
// to meet what L2 still holds; keeping the last 64 MB of the norm pass there by
// eviction hints won 3% on bf16 lists and lost 2% on fp32 ones, so there are
// none. In place, a coefficient of 1 ends the second pass at once.
//
// The list travels in the kernel's parameters (at most kMaxSegs tensors a
// launch), so a call uploads nothing, keeps nothing and can be captured.
//
// A thread adds a chunk's elements in fp32 and joins chunks in double. A
// partial sum outside [2^-96, 2^120], or not finite, is formed again in
// double from the registers: squares over- or underflow fp32 long before the
// norm does.

#include <algorithm>
#include <new>
#include <vector>

#include "common.cuh"
#include "internal.h"

namespace muon {

namespace {

constexpr int GC_THREADS = 256;
constexpr int GC_VEC = 8;
constexpr int GC_STEP = GC_THREADS * GC_VEC;  // 2048 elements: one group a thread
// Groups a thread takes of a chunk: 8 (128 bytes of bf16 in flight a thread),
// or 1 for lists too short to fill the GPU with such chunks.
constexpr int GC_ITERS = 8;
constexpr int kMaxSegs = 1024;
constexpr int kBlocksPerSm = 3;                // 98 KB in flight an SM; with 4 or 5 the same or 3% slower
constexpr int kMaxBlocks = 148 * kBlocksPerSm;  // one wave; a partial each

template <int N>
struct ClipTable {  // chunk_begin, chunks: in the launch's chunk size
  const void* src[N];
  void* dst[N];
  int64_t numel[N];
  int32_t chunk_begin[N];
  uint8_t types[N];  // bit 0: src is bf16, bit 1: dst is bf16
  int32_t n;
  int32_t chunks;
};
static_assert(sizeof(ClipTable<kMaxSegs>) + 64 < 32764, "kernel parameter space");

template <int N>
__device__ __forceinline__ int find_clip_segment(const ClipTable<N>& t, int chunk) {
  int lo = 0, hi = t.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.chunk_begin[mid] <= chunk)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// A thread's groups of 8 elements (16 bytes of bf16, 32 of fp32) in flight
// together: 128 bytes either way.
template <bool kBf>
struct Batch {
  static constexpr int kGroups = kBf ? 8 : 4;
  static constexpr int kWords = kBf ? 1 : 2;
  uint4 raw[kGroups][kWords];

  // groups first, first + GC_THREADS, ...
  __device__ __forceinline__ void load(const void* src, int first) {
    const uint4* p = static_cast<const uint4*>(src) + first * kWords;
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
#pragma unroll
      for (int q = 0; q < kWords; ++q) raw[i][q] = p[i * GC_THREADS * kWords + q];
  }
};

template <bool kBf>
__device__ __forceinline__ void load_group(const void* src, int g, uint4 (&raw)[Batch<kBf>::kWords]) {
#pragma unroll
  for (int q = 0; q < Batch<kBf>::kWords; ++q) raw[q] = static_cast<const uint4*>(src)[g * Batch<kBf>::kWords + q];
}

template <bool kBf>
__device__ __forceinline__ void unpack(const uint4 (&raw)[Batch<kBf>::kWords], float (&v)[GC_VEC]) {
  if constexpr (kBf) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw[0]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = __bfloat1622float2(h[k]);
      v[2 * k] = f.x;
      v[2 * k + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      v[4 * q] = __uint_as_float(raw[q].x);
      v[4 * q + 1] = __uint_as_float(raw[q].y);
      v[4 * q + 2] = __uint_as_float(raw[q].z);
      v[4 * q + 3] = __uint_as_float(raw[q].w);
    }
  }
}

// Group `at` of dst = round(v * coef).
template <bool kBf>
__device__ __forceinline__ void store_group(void* dst, int at, const float (&v)[GC_VEC], float coef) {
  if constexpr (kBf) {
    uint4 raw;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = __floats2bfloat162_rn(v[2 * k] * coef, v[2 * k + 1] * coef);
    static_cast<uint4*>(dst)[at] = raw;
  } else {
    float4* p = static_cast<float4*>(dst) + at * 2;
    p[0] = make_float4(v[0] * coef, v[1] * coef, v[2] * coef, v[3] * coef);
    p[1] = make_float4(v[4] * coef, v[5] * coef, v[6] * coef, v[7] * coef);
  }
}

__device__ __forceinline__ float load_one(const void* src, bool bf, int64_t e) {
  return bf ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(src)[e])
            : reinterpret_cast<const float*>(src)[e];
}

__device__ __forceinline__ void store_one(void* dst, bool bf, int64_t e, float x) {
  if (bf)
    reinterpret_cast<__nv_bfloat16*>(dst)[e] = __float2bfloat16_rn(x);
  else
    reinterpret_cast<float*>(dst)[e] = x;
}

// Elements e, e + GC_THREADS, ... below n (0 past it): unaligned chunks and ends of tensors.
__device__ __forceinline__ void load_ones(const void* src, bool bf, int e, int n, float (&v)[GC_VEC]) {
#pragma unroll
  for (int k = 0; k < GC_VEC; ++k) v[k] = e + k * GC_THREADS < n ? load_one(src, bf, e + k * GC_THREADS) : 0.f;
}

__device__ __forceinline__ bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// maximum that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) { return a != a ? a : (b != b ? b : fmaxf(a, b)); }
__device__ __forceinline__ double max_nan(double a, double b) { return a != a ? a : (b != b ? b : fmax(a, b)); }

template <int kNorm>
__device__ __forceinline__ double join(double a, double b) {
  if constexpr (kNorm == MUON_NORM_INF)
    return max_nan(a, b);
  else
    return a + b;
}

// One thread's |g|^p over `count` values: fp32, or double where fp32 would lose them.
template <int kNorm, int kCount>
__device__ __forceinline__ double reduce_values(const float (&v)[kCount]) {
  float acc = 0.f;
#pragma unroll
  for (int i = 0; i < kCount; ++i) {
    if constexpr (kNorm == MUON_NORM_2)
      acc = fmaf(v[i], v[i], acc);
    else if constexpr (kNorm == MUON_NORM_1)
      acc += fabsf(v[i]);
    else
      acc = max_nan(acc, fabsf(v[i]));
  }
  if constexpr (kNorm == MUON_NORM_INF) return acc;
  if (acc >= 0x1p-96f && acc <= 0x1p120f) return acc;
  double wide = 0.0;
#pragma unroll
  for (int i = 0; i < kCount; ++i) {
    const double x = v[i];
    if constexpr (kNorm == MUON_NORM_2)
      wide += x * x;
    else
      wide += fabs(x);
  }
  return wide;
}

template <int kNorm>
__device__ __forceinline__ double block_join(double x, double* shared) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x = join<kNorm>(x, __shfl_xor_sync(0xffffffffu, x, off));
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = x;
  __syncthreads();
  x = shared[0];
#pragma unroll
  for (int w = 1; w < GC_THREADS / 32; ++w) x = join<kNorm>(x, shared[w]);
  return x;
}

// A whole long chunk.
template <int kNorm, bool kBf>
__device__ __forceinline__ double norm_chunk(const void* src, double total) {
#pragma unroll 1
  for (int g = threadIdx.x; g < GC_ITERS * GC_THREADS; g += Batch<kBf>::kGroups * GC_THREADS) {
    Batch<kBf> b;
    b.load(src, g);
#pragma unroll
    for (int i = 0; i < Batch<kBf>::kGroups; ++i) {
      float v[GC_VEC];
      unpack<kBf>(b.raw[i], v);
      total = join<kNorm>(total, reduce_values<kNorm, GC_VEC>(v));
    }
  }
  return total;
}

// The aligned groups of any chunk, one at a time.
template <int kNorm, bool kBf>
__device__ __forceinline__ double norm_groups(const void* src, int groups, double total) {
#pragma unroll 1
  for (int g = threadIdx.x; g < groups; g += GC_THREADS) {
    uint4 raw[Batch<kBf>::kWords];
    load_group<kBf>(src, g, raw);
    float v[GC_VEC];
    unpack<kBf>(raw, v);
    total = join<kNorm>(total, reduce_values<kNorm, GC_VEC>(v));
  }
  return total;
}

template <int kNorm, int N, int kIters>
__global__ void __launch_bounds__(GC_THREADS, kBlocksPerSm)
    list_norm_kernel(const __grid_constant__ ClipTable<N> t, double* __restrict__ partials) {
  constexpr int kChunk = kIters * GC_STEP;
  __shared__ double red[GC_THREADS / 32];
  allow_next();
  double total = 0.0;
  for (int chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
    const int s = find_clip_segment(t, chunk);
    const bool bf = t.types[s] & 1;
    const int64_t e0 = int64_t(chunk - t.chunk_begin[s]) * kChunk;
    const char* src = static_cast<const char*>(t.src[s]) + e0 * (bf ? 2 : 4);
    const int n = static_cast<int>(min(int64_t(kChunk), t.numel[s] - e0));
    int done = 0;
    if (aligned16(src)) {
      if (kIters > 1 && n == kChunk)
        total = bf ? norm_chunk<kNorm, true>(src, total) : norm_chunk<kNorm, false>(src, total);
      else
        total = bf ? norm_groups<kNorm, true>(src, n / GC_VEC, total)
                   : norm_groups<kNorm, false>(src, n / GC_VEC, total);
      done = n / GC_VEC * GC_VEC;
    }
    for (int e = done + threadIdx.x; e < n; e += GC_STEP) {
      float v[GC_VEC];
      load_ones(src, bf, e, n, v);
      total = join<kNorm>(total, reduce_values<kNorm, GC_VEC>(v));
    }
  }
  total = block_join<kNorm>(total, red);
  if (threadIdx.x == 0) partials[blockIdx.x] = total;
}

// The blocks' partials joined in a fixed order: every thread returns the norm.
template <int kNorm>
__device__ __forceinline__ float join_partials(const double* partials, int n, double* shared) {
  double x = 0.0;
  for (int i = threadIdx.x; i < n; i += GC_THREADS) x = join<kNorm>(x, partials[i]);
  x = block_join<kNorm>(x, shared);
  return static_cast<float>(kNorm == MUON_NORM_2 ? sqrt(x) : x);
}

__device__ __forceinline__ float join_partials(int kind, const double* partials, int n, double* shared) {
  if (kind == MUON_NORM_2) return join_partials<MUON_NORM_2>(partials, n, shared);
  if (kind == MUON_NORM_1) return join_partials<MUON_NORM_1>(partials, n, shared);
  return join_partials<MUON_NORM_INF>(partials, n, shared);
}

__global__ void __launch_bounds__(GC_THREADS) total_norm_kernel(int kind, const double* __restrict__ partials, int n,
                                                                float* __restrict__ total) {
  __shared__ double red[GC_THREADS / 32];
  const float x = join_partials(kind, partials, n, red);
  if (threadIdx.x == 0) *total = x;
}

// A whole long chunk, or any number of aligned groups one at a time.
template <bool kBf, bool kOutBf, bool kWhole>
__device__ __forceinline__ void scale_groups(const void* src, void* dst, int groups, float coef) {
  if constexpr (kWhole) {
#pragma unroll 1
    for (int g = threadIdx.x; g < GC_ITERS * GC_THREADS; g += Batch<kBf>::kGroups * GC_THREADS) {
      Batch<kBf> b;
      b.load(src, g);
#pragma unroll
      for (int i = 0; i < Batch<kBf>::kGroups; ++i) {
        float v[GC_VEC];
        unpack<kBf>(b.raw[i], v);
        store_group<kOutBf>(dst, g + i * GC_THREADS, v, coef);
      }
    }
  } else {
#pragma unroll 1
    for (int g = threadIdx.x; g < groups; g += GC_THREADS) {
      uint4 raw[Batch<kBf>::kWords];
      load_group<kBf>(src, g, raw);
      float v[GC_VEC];
      unpack<kBf>(raw, v);
      store_group<kOutBf>(dst, g, v, coef);
    }
  }
}

template <bool kWhole>
__device__ __forceinline__ void scale_groups(const void* src, bool sbf, void* dst, bool dbf, int groups, float coef) {
  if (sbf && dbf)
    scale_groups<true, true, kWhole>(src, dst, groups, coef);
  else if (sbf)
    scale_groups<true, false, kWhole>(src, dst, groups, coef);
  else if (dbf)
    scale_groups<false, true, kWhole>(src, dst, groups, coef);
  else
    scale_groups<false, false, kWhole>(src, dst, groups, coef);
}

template <int N, int kIters>
__global__ void __launch_bounds__(GC_THREADS, kBlocksPerSm)
    list_scale_kernel(const __grid_constant__ ClipTable<N> t, int kind, const double* partials, int n_partials,
                      float max_norm, float* total_out, const float* total_in) {
  constexpr int kChunk = kIters * GC_STEP;
  __shared__ double red[GC_THREADS / 32];
  wait_previous();
  float total;
  if (partials) {
    total = join_partials(kind, partials, n_partials, red);
    if (total_out && blockIdx.x == 0 && threadIdx.x == 0) *total_out = total;
  } else {
    total = *total_in;
  }
  const double ratio = double(max_norm) / (double(total) + 1e-6);
  const float coef = ratio > 1.0 ? 1.f : static_cast<float>(ratio);  // NaN stays NaN
  for (int chunk = t.chunks - 1 - int(blockIdx.x); chunk >= 0; chunk -= gridDim.x) {
    const int s = find_clip_segment(t, chunk);
    const void* src = t.src[s];
    void* dst = t.dst[s];
    if (src == dst && coef == 1.f) continue;
    const bool sbf = t.types[s] & 1, dbf = t.types[s] & 2;
    const int64_t e0 = int64_t(chunk - t.chunk_begin[s]) * kChunk;
    const int n = static_cast<int>(min(int64_t(kChunk), t.numel[s] - e0));
    src = static_cast<const char*>(src) + e0 * (sbf ? 2 : 4);
    dst = static_cast<char*>(dst) + e0 * (dbf ? 2 : 4);
    int done = 0;
    if (aligned16(src) && aligned16(dst)) {
      if (kIters > 1 && n == kChunk)
        scale_groups<true>(src, sbf, dst, dbf, 0, coef);
      else
        scale_groups<false>(src, sbf, dst, dbf, n / GC_VEC, coef);
      done = n / GC_VEC * GC_VEC;
    }
    for (int e = done + threadIdx.x; e < n; e += GC_STEP) {
      float v[GC_VEC];
      load_ones(src, sbf, e, n, v);
#pragma unroll
      for (int k = 0; k < GC_VEC; ++k)
        if (e + k * GC_THREADS < n) store_one(dst, dbf, e + k * GC_THREADS, v[k] * coef);
    }
  }
}

constexpr int64_t kMaxChunks = 0x3fffffff;  // of a whole list

int64_t chunks_of(int64_t numel, int iters) { return (numel + iters * GC_STEP - 1) / (iters * GC_STEP); }

int check_segs(const muon_clip_seg* segs, int64_t n, bool outputs) {
  if (n < 0 || (n > 0 && !segs)) return set_error(MUON_ERR_ARG, "null clip segment table or negative count");
  int64_t chunks = 0;
  for (int64_t i = 0; i < n; ++i) {
    const muon_clip_seg& s = segs[i];
    if (s.numel < 0 || s.numel > kMaxChunks * GC_STEP || (chunks += chunks_of(s.numel, GC_ITERS)) > kMaxChunks)
      return set_error(MUON_ERR_ARG, "clip segment sizes out of range");
    const int es = s.grad_dtype == MUON_BF16 ? 2 : 4;
    if ((s.grad_dtype != MUON_BF16 && s.grad_dtype != MUON_F32) ||
        (outputs && s.out_dtype != MUON_BF16 && s.out_dtype != MUON_F32))
      return set_error(MUON_ERR_ARG, "clip dtypes must be MUON_BF16 or MUON_F32");
    if (s.numel == 0) continue;
    if (!s.grad || (outputs && !s.out)) return set_error(MUON_ERR_ARG, "null clip segment pointer");
    if (reinterpret_cast<uintptr_t>(s.grad) % es ||
        (outputs && reinterpret_cast<uintptr_t>(s.out) % (s.out_dtype == MUON_BF16 ? 2 : 4)))
      return set_error(MUON_ERR_ARG, "clip segment pointer not aligned to its dtype");
    if (outputs && s.out == s.grad && s.out_dtype != s.grad_dtype)
      return set_error(MUON_ERR_ARG, "clipping in place needs one dtype");
  }
  return MUON_OK;
}

// Outputs must not share memory with one another, with another segment's
// gradient or with the norm: blocks read and write them in no fixed order.
int check_overlap(const muon_clip_seg* segs, int64_t n, const float* norm) try {
  struct Span {
    uintptr_t begin, end;
    int64_t seg;
  };
  std::vector<Span> outs;
  outs.reserve(n);
  for (int64_t i = 0; i < n; ++i) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(segs[i].out);
    if (segs[i].numel > 0) outs.push_back({p, p + segs[i].numel * (segs[i].out_dtype == MUON_BF16 ? 2 : 4), i});
  }
  std::sort(outs.begin(), outs.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
  for (size_t i = 1; i < outs.size(); ++i)
    if (outs[i].begin < outs[i - 1].end) return set_error(MUON_ERR_ARG, "clipped gradients overlap in memory");
  auto written = [&outs](const void* p, uintptr_t bytes) {
    const uintptr_t begin = reinterpret_cast<uintptr_t>(p), end = begin + bytes;
    auto after =
        std::lower_bound(outs.begin(), outs.end(), end, [](const Span& s, uintptr_t e) { return s.begin < e; });
    return after != outs.begin() && (after - 1)->end > begin;
  };
  for (int64_t i = 0; i < n; ++i) {
    if (segs[i].numel == 0 || segs[i].grad == segs[i].out) continue;
    if (written(segs[i].grad, segs[i].numel * (segs[i].grad_dtype == MUON_BF16 ? 2 : 4)))
      return set_error(MUON_ERR_ARG, "gradients overlap the memory they are clipped into");
  }
  if (written(norm, sizeof(float))) return set_error(MUON_ERR_ARG, "the norm overlaps the clipped gradients");
  return MUON_OK;
} catch (const std::bad_alloc&) {
  return set_error(MUON_ERR_ARG, "out of host memory");
}

// Fills `t` with segments from `i` on (empty ones skipped) and returns the next index.
template <int N>
int64_t fill_table(ClipTable<N>& t, const muon_clip_seg* segs, int64_t i, int64_t n, int iters) {
  t.n = 0;
  int64_t chunks = 0;
  for (; i < n && t.n < N; ++i) {
    const muon_clip_seg& s = segs[i];
    if (s.numel == 0) continue;
    t.src[t.n] = s.grad;
    t.dst[t.n] = s.out;
    t.numel[t.n] = s.numel;
    t.chunk_begin[t.n] = static_cast<int32_t>(chunks);
    t.types[t.n] = (s.grad_dtype == MUON_BF16 ? 1 : 0) | (s.out_dtype == MUON_BF16 ? 2 : 0);
    ++t.n;
    chunks += chunks_of(s.numel, iters);
  }
  t.chunks = static_cast<int32_t>(chunks);
  return i;
}

int blocks_for(int chunks) { return chunks < kMaxBlocks ? chunks : kMaxBlocks; }

// How a list is launched: its parameter block is copied with every launch, so
// short lists take a short one.
constexpr int kShortSegs = 64;

// Long chunks once they give every resident block two.
int iters_for(const muon_clip_seg* segs, int64_t n) {
  int64_t chunks = 0;
  for (int64_t i = 0; i < n; ++i) chunks += chunks_of(segs[i].numel, GC_ITERS);
  return chunks >= 2 * kMaxBlocks ? GC_ITERS : 1;
}

// Runs launch(table) for every batch of the list.
template <int N, int kIters, typename F>
int for_batches(const muon_clip_seg* segs, int64_t n, F&& launch) {
  ClipTable<N> t;
  for (int64_t i = 0; i < n;) {
    i = fill_table(t, segs, i, n, kIters);
    if (t.n == 0) break;
    const int rc = launch(t);
    if (rc != MUON_OK) return rc;
  }
  return MUON_OK;
}

template <int N, int kIters>
int norm_batches(const muon_clip_seg* segs, int64_t n, int kind, double* partials, int* n_partials,
                 cudaStream_t stream) {
  *n_partials = 0;
  return for_batches<N, kIters>(segs, n, [&](const ClipTable<N>& t) {
    const int blocks = blocks_for(t.chunks);
    double* out = partials + *n_partials;
    if (kind == MUON_NORM_2)
      list_norm_kernel<MUON_NORM_2, N, kIters><<<blocks, GC_THREADS, 0, stream>>>(t, out);
    else if (kind == MUON_NORM_1)
      list_norm_kernel<MUON_NORM_1, N, kIters><<<blocks, GC_THREADS, 0, stream>>>(t, out);
    else
      list_norm_kernel<MUON_NORM_INF, N, kIters><<<blocks, GC_THREADS, 0, stream>>>(t, out);
    *n_partials += blocks;
    return check_cuda(cudaGetLastError(), "list norm launch");
  });
}

template <int N, int kIters>
int scale_batches(const muon_clip_seg* segs, int64_t n, int kind, const double* partials, int n_partials,
                  float max_norm, float* total_out, const float* total_in, cudaStream_t stream) {
  return for_batches<N, kIters>(segs, n, [&](const ClipTable<N>& t) {
    const int rc = launch_overlapped("list scale launch", list_scale_kernel<N, kIters>, blocks_for(t.chunks),
                                     GC_THREADS, stream, t, kind, partials, n_partials, max_norm, total_out, total_in);
    total_out = nullptr;  // written by the first batch
    return rc;
  });
}

int norm_list(const muon_clip_seg* segs, int64_t n, int kind, double* partials, int* n_partials, cudaStream_t stream) {
  const bool lng = iters_for(segs, n) == GC_ITERS;
  if (n <= kShortSegs)
    return lng ? norm_batches<kShortSegs, GC_ITERS>(segs, n, kind, partials, n_partials, stream)
               : norm_batches<kShortSegs, 1>(segs, n, kind, partials, n_partials, stream);
  return lng ? norm_batches<kMaxSegs, GC_ITERS>(segs, n, kind, partials, n_partials, stream)
             : norm_batches<kMaxSegs, 1>(segs, n, kind, partials, n_partials, stream);
}

int scale_list(const muon_clip_seg* segs, int64_t n, int kind, const double* partials, int n_partials, float max_norm,
               float* total_out, const float* total_in, cudaStream_t stream) {
  const bool lng = iters_for(segs, n) == GC_ITERS;
  auto run = [&](auto batches) {
    return batches(segs, n, kind, partials, n_partials, max_norm, total_out, total_in, stream);
  };
  if (n <= kShortSegs) return lng ? run(scale_batches<kShortSegs, GC_ITERS>) : run(scale_batches<kShortSegs, 1>);
  return lng ? run(scale_batches<kMaxSegs, GC_ITERS>) : run(scale_batches<kMaxSegs, 1>);
}

bool all_empty(const muon_clip_seg* segs, int64_t n) {
  for (int64_t i = 0; i < n; ++i)
    if (segs[i].numel != 0) return false;
  return true;
}

}  // namespace

int64_t clip_workspace_bytes(int64_t n_segs) {
  if (n_segs < 0 || n_segs > (int64_t(1) << 30)) return -1;
  const int64_t batches = n_segs / kMaxSegs + 1;
  return batches * kMaxBlocks * int64_t(sizeof(double));
}

int launch_total_norm(const muon_clip_seg* segs, int64_t n_segs, int norm_kind, void* workspace, float* total,
                      cudaStream_t stream) {
  if (norm_kind < MUON_NORM_2 || norm_kind > MUON_NORM_INF) return set_error(MUON_ERR_ARG, "unknown norm kind");
  if (!total || misaligned(total, 4) || !workspace || misaligned(workspace, 16))
    return set_error(MUON_ERR_ARG, "norm output or workspace missing or misaligned");
  if (int rc = check_segs(segs, n_segs, false)) return rc;
  double* partials = static_cast<double*>(workspace);
  int n = 0;
  if (int rc = norm_list(segs, n_segs, norm_kind, partials, &n, stream)) return rc;
  total_norm_kernel<<<1, GC_THREADS, 0, stream>>>(norm_kind, partials, n, total);
  return check_cuda(cudaGetLastError(), "total norm launch");
}

int launch_clip_grads(const muon_clip_seg* segs, int64_t n_segs, int norm_kind, float max_norm, void* workspace,
                      float* total, cudaStream_t stream) {
  if (int rc = check_segs(segs, n_segs, true)) return rc;
  if (int rc = check_overlap(segs, n_segs, total)) return rc;
  if (all_empty(segs, n_segs)) return launch_total_norm(segs, n_segs, norm_kind, workspace, total, stream);
  if (norm_kind < MUON_NORM_2 || norm_kind > MUON_NORM_INF) return set_error(MUON_ERR_ARG, "unknown norm kind");
  if (!total || misaligned(total, 4) || !workspace || misaligned(workspace, 16))
    return set_error(MUON_ERR_ARG, "norm output or workspace missing or misaligned");
  double* partials = static_cast<double*>(workspace);
  int n = 0;
  if (int rc = norm_list(segs, n_segs, norm_kind, partials, &n, stream)) return rc;
  return scale_list(segs, n_segs, norm_kind, partials, n, max_norm, total, nullptr, stream);
}

int launch_scale_grads(const muon_clip_seg* segs, int64_t n_segs, float max_norm, const float* total,
                       cudaStream_t stream) {
  if (!total || misaligned(total, 4)) return set_error(MUON_ERR_ARG, "norm missing or misaligned");
  if (int rc = check_segs(segs, n_segs, true)) return rc;
  if (int rc = check_overlap(segs, n_segs, total)) return rc;
  return scale_list(segs, n_segs, 0, nullptr, 0, max_norm, nullptr, total, stream);
}

}  // namespace muon
