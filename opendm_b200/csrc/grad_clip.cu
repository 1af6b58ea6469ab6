// Norm of a list of gradients, and clipping in place or into other tensors.
//
//   total = (sum |g|^p)^(1/p), p = 1, 2, inf;  coef = min(max_norm / (total + 1e-6), 1)
//   out   = round(g * coef)
//
// Two launches: the norm pass leaves one double per block, the scale pass
// adds those (every block the same sum in the same order) and rescales. HBM
// bound: one read for the norm, one read and one write for the scaling; the
// scale pass walks the list backwards, so what the norm pass read last is
// still in L2. In place, a coefficient of 1 ends the second pass at once.
//
// The list travels in the kernel's parameters (at most kMaxSegs tensors a
// launch), so a call uploads nothing, keeps nothing and can be captured.
//
// A thread adds a chunk's elements in fp32 and joins chunks in double. A
// partial sum outside [2^-96, 2^120], or not finite, is formed again in
// double from the registers: squares over- or underflow fp32 long before the
// norm does.

#include <cmath>

#include "common.cuh"
#include "internal.h"

namespace muon {

namespace {

constexpr int GC_THREADS = 256;
constexpr int GC_VEC = 8;
constexpr int GC_ITERS = 8;
constexpr int64_t GC_CHUNK = int64_t(GC_THREADS) * GC_VEC * GC_ITERS;  // 16384
constexpr int kMaxSegs = 1024;
constexpr int kMaxBlocks = 148 * 8;  // partials per launch

template <int N>
struct ClipTable {
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

__device__ __forceinline__ void load_group(const void* src, bool bf, int64_t e, float (&v)[GC_VEC]) {
  if (bf) {
    const uint4 raw = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(src) + e);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(h[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(src) + e);
    const float4 a = p[0], b = p[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
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

template <int kNorm, int N>
__global__ void __launch_bounds__(GC_THREADS) list_norm_kernel(const __grid_constant__ ClipTable<N> t,
                                                               double* __restrict__ partials) {
  __shared__ double red[GC_THREADS / 32];
  double total = 0.0;
  for (int chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
    const int s = find_clip_segment(t, chunk);
    const void* src = t.src[s];
    const int64_t numel = t.numel[s];
    const bool bf = t.types[s] & 1;
    const int64_t e0 = int64_t(chunk - t.chunk_begin[s]) * GC_CHUNK;
    const int64_t e1 = min(e0 + GC_CHUNK, numel);
    int64_t done = e0;
    if (aligned16(src)) {
      done = e0 + (e1 - e0) / GC_VEC * GC_VEC;
      float v[4][GC_VEC];
#pragma unroll
      for (int half = 0; half < GC_ITERS / 4; ++half) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t e = e0 + (int64_t(half * 4 + i) * GC_THREADS + threadIdx.x) * GC_VEC;
          if (e < done) {
            load_group(src, bf, e, v[i]);
          } else {
#pragma unroll
            for (int k = 0; k < GC_VEC; ++k) v[i][k] = 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) total = join<kNorm>(total, reduce_values<kNorm, GC_VEC>(v[i]));
      }
    }
    for (int64_t e = done + threadIdx.x; e < e1; e += GC_THREADS) {
      const float v[1] = {load_one(src, bf, e)};
      total = join<kNorm>(total, reduce_values<kNorm, 1>(v));
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

template <int N>
__global__ void __launch_bounds__(GC_THREADS) list_scale_kernel(const __grid_constant__ ClipTable<N> t, int kind,
                                                                const double* __restrict__ partials, int n_partials,
                                                                float max_norm, float* __restrict__ total_out,
                                                                const float* __restrict__ total_in) {
  __shared__ double red[GC_THREADS / 32];
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
    const int64_t numel = t.numel[s];
    const bool sbf = t.types[s] & 1, dbf = t.types[s] & 2;
    const int64_t e0 = int64_t(chunk - t.chunk_begin[s]) * GC_CHUNK;
    const int64_t e1 = min(e0 + GC_CHUNK, numel);
    int64_t done = e0;
    if (aligned16(src) && aligned16(dst)) {
      done = e0 + (e1 - e0) / GC_VEC * GC_VEC;
      float v[4][GC_VEC];
#pragma unroll
      for (int half = 0; half < GC_ITERS / 4; ++half) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t e = e0 + (int64_t(half * 4 + i) * GC_THREADS + threadIdx.x) * GC_VEC;
          if (e < done) load_group(src, sbf, e, v[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t e = e0 + (int64_t(half * 4 + i) * GC_THREADS + threadIdx.x) * GC_VEC;
          if (e >= done) continue;
          if (dbf) {
            uint4 raw;
            __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
            for (int k = 0; k < 4; ++k) h[k] = __floats2bfloat162_rn(v[i][2 * k] * coef, v[i][2 * k + 1] * coef);
            *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(dst) + e) = raw;
          } else {
            float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(dst) + e);
            p[0] = make_float4(v[i][0] * coef, v[i][1] * coef, v[i][2] * coef, v[i][3] * coef);
            p[1] = make_float4(v[i][4] * coef, v[i][5] * coef, v[i][6] * coef, v[i][7] * coef);
          }
        }
      }
    }
    for (int64_t e = done + threadIdx.x; e < e1; e += GC_THREADS)
      store_one(dst, dbf, e, load_one(src, sbf, e) * coef);
  }
}

constexpr int64_t kMaxChunks = 0x3fffffff;  // of a whole list

int64_t chunks_of(int64_t numel) { return (numel + GC_CHUNK - 1) / GC_CHUNK; }

int check_segs(const muon_clip_seg* segs, int64_t n, bool outputs) {
  if (n < 0 || (n > 0 && !segs)) return set_error(MUON_ERR_ARG, "null clip segment table or negative count");
  int64_t chunks = 0;
  for (int64_t i = 0; i < n; ++i) {
    const muon_clip_seg& s = segs[i];
    if (s.numel < 0 || s.numel > GC_CHUNK * kMaxChunks || (chunks += chunks_of(s.numel)) > kMaxChunks)
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

// Fills `t` with segments from `i` on (empty ones skipped) and returns the next index.
template <int N>
int64_t fill_table(ClipTable<N>& t, const muon_clip_seg* segs, int64_t i, int64_t n) {
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
    chunks += chunks_of(s.numel);
  }
  t.chunks = static_cast<int32_t>(chunks);
  return i;
}

int blocks_for(int chunks) { return chunks < kMaxBlocks ? chunks : kMaxBlocks; }

// Runs `launch(table)` for every batch of the list.
template <int N, typename F>
int for_batches(const muon_clip_seg* segs, int64_t n, F&& launch) {
  ClipTable<N> t;
  for (int64_t i = 0; i < n;) {
    i = fill_table(t, segs, i, n);
    if (t.n == 0) break;
    const int rc = launch(t);
    if (rc != MUON_OK) return rc;
  }
  return MUON_OK;
}

template <int N>
int norm_batches(const muon_clip_seg* segs, int64_t n, int kind, double* partials, int* n_partials,
                 cudaStream_t stream) {
  *n_partials = 0;
  return for_batches<N>(segs, n, [&](const ClipTable<N>& t) {
    const int blocks = blocks_for(t.chunks);
    double* out = partials + *n_partials;
    if (kind == MUON_NORM_2)
      list_norm_kernel<MUON_NORM_2, N><<<blocks, GC_THREADS, 0, stream>>>(t, out);
    else if (kind == MUON_NORM_1)
      list_norm_kernel<MUON_NORM_1, N><<<blocks, GC_THREADS, 0, stream>>>(t, out);
    else
      list_norm_kernel<MUON_NORM_INF, N><<<blocks, GC_THREADS, 0, stream>>>(t, out);
    *n_partials += blocks;
    return check_cuda(cudaGetLastError(), "list norm launch");
  });
}

template <int N>
int scale_batches(const muon_clip_seg* segs, int64_t n, int kind, const double* partials, int n_partials,
                  float max_norm, float* total_out, const float* total_in, cudaStream_t stream) {
  return for_batches<N>(segs, n, [&](const ClipTable<N>& t) {
    list_scale_kernel<N><<<blocks_for(t.chunks), GC_THREADS, 0, stream>>>(t, kind, partials, n_partials, max_norm,
                                                                         total_out, total_in);
    total_out = nullptr;  // written by the first batch
    return check_cuda(cudaGetLastError(), "list scale launch");
  });
}

// The parameter block is copied with every launch: short lists take a short one.
constexpr int kShortSegs = 64;

int norm_list(const muon_clip_seg* segs, int64_t n, int kind, double* partials, int* n_partials, cudaStream_t stream) {
  return n <= kShortSegs ? norm_batches<kShortSegs>(segs, n, kind, partials, n_partials, stream)
                         : norm_batches<kMaxSegs>(segs, n, kind, partials, n_partials, stream);
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
  if (!total || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u))
    return set_error(MUON_ERR_ARG, "null norm output, or workspace missing or misaligned");
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
  if (all_empty(segs, n_segs)) return launch_total_norm(segs, n_segs, norm_kind, workspace, total, stream);
  if (norm_kind < MUON_NORM_2 || norm_kind > MUON_NORM_INF) return set_error(MUON_ERR_ARG, "unknown norm kind");
  if (!total || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u))
    return set_error(MUON_ERR_ARG, "null norm output, or workspace missing or misaligned");
  double* partials = static_cast<double*>(workspace);
  int n = 0;
  if (int rc = norm_list(segs, n_segs, norm_kind, partials, &n, stream)) return rc;
  return n_segs <= kShortSegs
             ? scale_batches<kShortSegs>(segs, n_segs, norm_kind, partials, n, max_norm, total, nullptr, stream)
             : scale_batches<kMaxSegs>(segs, n_segs, norm_kind, partials, n, max_norm, total, nullptr, stream);
}

int launch_scale_grads(const muon_clip_seg* segs, int64_t n_segs, float max_norm, const float* total,
                       cudaStream_t stream) {
  if (!total) return set_error(MUON_ERR_ARG, "null norm");
  if (int rc = check_segs(segs, n_segs, true)) return rc;
  return n_segs <= kShortSegs
             ? scale_batches<kShortSegs>(segs, n_segs, 0, nullptr, 0, max_norm, nullptr, total, stream)
             : scale_batches<kMaxSegs>(segs, n_segs, 0, nullptr, 0, max_norm, nullptr, total, stream);
}

}  // namespace muon
