// Fused AdamW for the reference's non-Muon parameter group.
// Reference: _adamw_step / _call_adamw_functional (opendm/optimizer/
// muon_adamw.py:131-175, :333-343), which calls torch.optim.adamw's
// single-tensor path (decoupled weight decay) once per parameter. Here every
// parameter of the group is one segment of a single launch and each element
// is read and written once:
//   p = p * (1 - lr*wd)                      (rounded to the param dtype)
//   m = m + (1 - beta1) * (g - m)            (lerp, fused multiply-add)
//   v = fl(v * beta2) + fl(fl((1-beta2) * g) * g)
//   p = p + (-step_size) * (m / (fl(sqrt(v) / bc2_sqrt) + eps))
// The rounding sequence follows torch's CPU kernels for these ops.

#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "internal.h"

namespace muon {

constexpr int ADAM_THREADS = 256;
constexpr int ADAM_VEC = 4;
constexpr int ADAM_ITERS = 8;
constexpr int64_t ADAM_CHUNK = int64_t(ADAM_THREADS) * ADAM_VEC * ADAM_ITERS;  // 8192

int64_t adamw_chunks(int64_t numel) { return numel <= 0 ? 0 : (numel + ADAM_CHUNK - 1) / ADAM_CHUNK; }

__device__ __forceinline__ int find_adam_segment(const muon_adamw_seg* segs, int n_segs, int64_t chunk) {
  int lo = 0, hi = n_segs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (segs[mid].chunk_begin <= chunk)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float decayed(float p, float wd_factor, bool bf16_param) {
  return bf16_param ? bf16_round(p * wd_factor) : p * wd_factor;
}

__device__ __forceinline__ float adam_elem(float p, float g, float& m, float& v, float beta1w, float beta2,
                                           float one_minus_beta2, float eps, float wd_factor, float neg_step,
                                           float bc2_sqrt, bool bf16_param) {
  if (wd_factor != 1.f) p = decayed(p, wd_factor, bf16_param);
  m = fmaf(beta1w, g - m, m);
  v = __fadd_rn(__fmul_rn(v, beta2), __fmul_rn(__fmul_rn(one_minus_beta2, g), g));
  const float denom = __fadd_rn(__fdiv_rn(sqrtf(v), bc2_sqrt), eps);
  return __fadd_rn(p, __fmul_rn(neg_step, __fdiv_rn(m, denom)));
}

// Gradient-norm clipping folded into the read (clip.cu): g' = g * coef with
// the coefficient and the product in the gradient's dtype (torch's CUDA
// _foreach_mul_ with a 0-d coefficient tensor).
__device__ __forceinline__ float clip_grad_adam(float g, float coef, bool bf) {
  return bf ? bf16_round(g * bf16_round(coef)) : g * coef;
}

__global__ void __launch_bounds__(ADAM_THREADS) adamw_kernel(const muon_adamw_seg* __restrict__ segs, int n_segs,
                                                             float beta1w, float beta2, float one_minus_beta2,
                                                             float eps, float wd_factor,
                                                             const float* __restrict__ grad_scale) {
  const int64_t chunk = blockIdx.x;
  const muon_adamw_seg sg = segs[find_adam_segment(segs, n_segs, chunk)];
  const int64_t e0 = (chunk - sg.chunk_begin) * ADAM_CHUNK;
  const int64_t e1 = min(e0 + ADAM_CHUNK, sg.numel);
  const bool pbf = sg.param_dtype == MUON_BF16;
  const bool gbf = sg.grad_dtype == MUON_BF16;
  const float neg_step = -sg.step_size;
  const bool vec_ok = (sg.numel % 4) == 0 &&
                      ((reinterpret_cast<uintptr_t>(sg.param) | reinterpret_cast<uintptr_t>(sg.grad) |
                        reinterpret_cast<uintptr_t>(sg.exp_avg) | reinterpret_cast<uintptr_t>(sg.exp_avg_sq)) &
                       15u) == 0;
  if (vec_ok) {
    for (int it = 0; it < ADAM_ITERS; ++it) {
      const int64_t e = e0 + (int64_t(it) * ADAM_THREADS + threadIdx.x) * ADAM_VEC;
      if (e >= e1) break;
      float p[4], g[4];
      if (pbf) {
        const uint2 raw = *reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(sg.param) + e);
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
        const float2 a = __bfloat1622float2(h[0]), b = __bfloat1622float2(h[1]);
        p[0] = a.x, p[1] = a.y, p[2] = b.x, p[3] = b.y;
      } else {
        const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sg.param) + e);
        p[0] = a.x, p[1] = a.y, p[2] = a.z, p[3] = a.w;
      }
      if (gbf) {
        const uint2 raw = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(sg.grad) + e));
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
        const float2 a = __bfloat1622float2(h[0]), b = __bfloat1622float2(h[1]);
        g[0] = a.x, g[1] = a.y, g[2] = b.x, g[3] = b.y;
      } else {
        const float4 a = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sg.grad) + e));
        g[0] = a.x, g[1] = a.y, g[2] = a.z, g[3] = a.w;
      }
      if (grad_scale != nullptr) {
        const float coef = *grad_scale;
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = clip_grad_adam(g[i], coef, gbf);
      }
      float4 m4 = *reinterpret_cast<float4*>(sg.exp_avg + e);
      float4 v4 = *reinterpret_cast<float4*>(sg.exp_avg_sq + e);
      float m[4] = {m4.x, m4.y, m4.z, m4.w}, v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        p[i] = adam_elem(p[i], g[i], m[i], v[i], beta1w, beta2, one_minus_beta2, eps, wd_factor, neg_step,
                         sg.bc2_sqrt, pbf);
      *reinterpret_cast<float4*>(sg.exp_avg + e) = make_float4(m[0], m[1], m[2], m[3]);
      *reinterpret_cast<float4*>(sg.exp_avg_sq + e) = make_float4(v[0], v[1], v[2], v[3]);
      if (pbf) {
        uint2 raw;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
        h[0] = __floats2bfloat162_rn(p[0], p[1]);
        h[1] = __floats2bfloat162_rn(p[2], p[3]);
        *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(sg.param) + e) = raw;
      } else {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(sg.param) + e) = make_float4(p[0], p[1], p[2], p[3]);
      }
    }
  } else {
    for (int64_t e = e0 + threadIdx.x; e < e1; e += ADAM_THREADS) {
      float p = pbf ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(sg.param)[e])
                    : reinterpret_cast<const float*>(sg.param)[e];
      float g = gbf ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(sg.grad)[e])
                    : reinterpret_cast<const float*>(sg.grad)[e];
      if (grad_scale != nullptr) g = clip_grad_adam(g, *grad_scale, gbf);
      float m = sg.exp_avg[e], v = sg.exp_avg_sq[e];
      p = adam_elem(p, g, m, v, beta1w, beta2, one_minus_beta2, eps, wd_factor, neg_step, sg.bc2_sqrt, pbf);
      sg.exp_avg[e] = m;
      sg.exp_avg_sq[e] = v;
      if (pbf)
        reinterpret_cast<__nv_bfloat16*>(sg.param)[e] = __float2bfloat16_rn(p);
      else
        reinterpret_cast<float*>(sg.param)[e] = p;
    }
  }
}

// ------------------------------------------------------------ row gradients
// The same update of a [rows][dim] parameter whose gradient is zero outside
// the rows listed in ids (ascending). A block takes 4096 consecutive
// elements, finds the listed rows among its own by a 32-way search of ids and
// keeps their slots in shared memory; elements of the other rows take g = 0,
// so the results equal adamw_kernel's on the dense gradient, at the bytes of
// param and moments plus those of the listed rows.
template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
  if constexpr (sizeof(T) == 2) {
    const uint2 raw = *reinterpret_cast<const uint2*>(p);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
    const float2 a = __bfloat1622float2(h[0]), b = __bfloat1622float2(h[1]);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  } else {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
  if constexpr (sizeof(T) == 2) {
    uint2 raw;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
    h[0] = __floats2bfloat162_rn(v[0], v[1]);
    h[1] = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) = raw;
  } else {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
}
template <typename T>
__device__ __forceinline__ float load1(const T* p) {
  if constexpr (sizeof(T) == 2)
    return __bfloat162float(*p);
  else
    return *p;
}
template <typename T>
__device__ __forceinline__ void store1(T* p, float v) {
  if constexpr (sizeof(T) == 2)
    *p = __float2bfloat16_rn(v);
  else
    *p = v;
}

// First index in ids[0, n) with ids[index] >= row, by a whole warp: 32
// probes a step, so four dependent loads for a million rows.
__device__ __forceinline__ int64_t warp_lower_bound(const int64_t* ids, int64_t n, int64_t row) {
  const int lane = threadIdx.x & 31;
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t step = (hi - lo + 31) / 32;
    const int64_t at = lo + int64_t(lane) * step;
    const bool below = at < hi && ids[at] < row;
    const int k = __popc(__ballot_sync(0xffffffffu, below));  // the probes below `row` come first
    if (k == 0) return lo;
    const int64_t last_below = lo + int64_t(k - 1) * step;
    hi = min(hi, last_below + step);
    lo = last_below + 1;
  }
  return lo;
}

struct AdamwRowsArgs {
  float* exp_avg;
  float* exp_avg_sq;
  const int64_t* ids;
  const int64_t* count;
  int64_t rows, dim, cap, numel;
  float beta1w, beta2, one_minus_beta2, eps, wd_factor, neg_step, bc2_sqrt;
  const float* grad_scale;
  bool quiet;
};

// Rows that no step has touched, or none for many steps, keep zero or denormal
// first moments, whose division is a slow one. With |m| <= 2^-90 after the
// step, eps >= 2^-30 and a step size of at most 2^6 the update is at most
// 2^-54: for |p| >= 2^-20 under a quarter of p's last place, so p stays as it
// is (and for m = 0 any p does); only the moments decay, and zeros stay put.
constexpr float kQuietMoment = 0x1p-90f, kQuietParam = 0x1p-20f;

constexpr int ROWS_ITERS = 4;
constexpr int ROWS_BLOCKS = 8;  // 64 warps an SM: the element's two divisions and root fill the issue slots
constexpr int ROWS_CHUNK = ADAM_THREADS * ADAM_VEC * ROWS_ITERS;  // 4096 elements of a block

// kVector: param and moments are 16-byte aligned; four consecutive elements
// may span rows. kGradVector: they never do, and rows of values are aligned too.
// 151936 x 2048 bf16, 16384 tokens: 999 us (6.26 TB/s of 6.55 measured); with
// 8192 elements a block 991, with 2048 1079, with six blocks an SM 1034. An fp32
// 32003 x 257: 54 us with 2048 or 4096, 57 with 8192; a division of integers and
// a slot lookup for each group of four, and 2009 blocks in 1184 places, are what
// it has over the first. With zero moments in the 95% of its rows no token names
// (the start of a run) the first takes 694 us, the dense kernel, whose divisions
// are then slow ones, 1382.
template <typename P, typename G, bool kVector, bool kGradVector>
__global__ void __launch_bounds__(ADAM_THREADS, ROWS_BLOCKS)
    adamw_rows_kernel(P* __restrict__ param, const G* __restrict__ values, const AdamwRowsArgs a) {
  // slot of each of the block's rows (at most ROWS_CHUNK + 1, when dim is 1), or -1
  extern __shared__ int32_t slots[];
  const int64_t e0 = int64_t(blockIdx.x) * ROWS_CHUNK;
  const int len = static_cast<int>(min(int64_t(ROWS_CHUNK), a.numel - e0));
  const int64_t row0 = e0 / a.dim, row1 = (e0 + len - 1) / a.dim + 1;
  const uint32_t col0 = static_cast<uint32_t>(e0 - row0 * a.dim), dim = static_cast<uint32_t>(a.dim);
  const int body = kVector ? len / ADAM_VEC * ADAM_VEC : 0;
  // whether the block looks quiet, by one first moment a thread: the loop below that tests every group for it
  // would cost the others registers
  const float probe = kVector && int(threadIdx.x) * ADAM_VEC < body ? a.exp_avg[e0 + threadIdx.x * ADAM_VEC] : 0.f;
  const int n_rows = static_cast<int>(row1 - row0);
  for (int r = threadIdx.x; r < n_rows; r += ADAM_THREADS) slots[r] = -1;
  __syncthreads();
  if (threadIdx.x < 32) {
    const int64_t n = a.count ? min(max(*a.count, int64_t(0)), a.cap) : a.cap;
    const int64_t first = warp_lower_bound(a.ids, n, row0);
    for (int64_t i = first + threadIdx.x;; i += 32) {
      const int64_t id = i < n ? a.ids[i] : row1;
      const bool mine = id >= row0 && id < row1;
      if (mine) slots[id - row0] = static_cast<int32_t>(i);
      if (!__all_sync(0xffffffffu, mine)) break;
    }
  }
  const bool pbf = sizeof(P) == 2, gbf = sizeof(G) == 2;
  const float coef = a.grad_scale ? *a.grad_scale : 1.f;
  auto clipped = [&](float g) { return a.grad_scale ? clip_grad_adam(g, coef, gbf) : g; };
  const float unlisted = clipped(0.f);  // 0, or NaN with a NaN or infinite coefficient, as in the dense form
  const bool mostly_quiet = __syncthreads_and(a.quiet && unlisted == 0.f && fabsf(probe) <= kQuietMoment);
  auto element = [&](int o) {  // gradient of element o of the block
    const uint32_t at = col0 + o, r = at / dim;
    const int32_t slot = slots[r];
    return slot < 0 ? unlisted : clipped(load1(values + int64_t(slot) * a.dim + (at - r * dim)));
  };
  auto update = [&](float& p, float g, float& m, float& v) {
    p = adam_elem(p, g, m, v, a.beta1w, a.beta2, a.one_minus_beta2, a.eps, a.wd_factor, a.neg_step, a.bc2_sqrt, pbf);
  };
  auto sweep = [&](auto look_for_quiet) {
    constexpr bool kQuiet = decltype(look_for_quiet)::value;
    for (int o = threadIdx.x * ADAM_VEC; o < body; o += ADAM_THREADS * ADAM_VEC) {
      float p[4], m[4], v[4];
      load4(param + e0 + o, p);
      load4(a.exp_avg + e0 + o, m);
      load4(a.exp_avg_sq + e0 + o, v);
      float g[4] = {unlisted, unlisted, unlisted, unlisted};
      const uint32_t at = col0 + o, r = at / dim, col = at - r * dim;
      if (kGradVector || col + 3 < dim) {
        const int32_t slot = slots[r];
        if constexpr (kQuiet) {
          if (slot < 0) {
            bool quiet = true;
            uint32_t changed = 0;
            float np[4], nm[4], nv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              np[i] = a.wd_factor != 1.f ? decayed(p[i], a.wd_factor, pbf) : p[i];
              nm[i] = fmaf(a.beta1w, 0.f - m[i], m[i]);
              nv[i] = __fmul_rn(v[i], a.beta2);
              quiet = quiet && fabsf(nm[i]) <= kQuietMoment && v[i] >= 0.f &&
                      (nm[i] == 0.f || fabsf(np[i]) >= kQuietParam);
              changed |= (__float_as_uint(nm[i]) ^ __float_as_uint(m[i])) |
                         (__float_as_uint(nv[i]) ^ __float_as_uint(v[i]));
            }
            if (quiet) {
              if (changed) {
                store4(a.exp_avg + e0 + o, nm);
                store4(a.exp_avg_sq + e0 + o, nv);
              }
              if (a.wd_factor != 1.f) store4(param + e0 + o, np);
              continue;
            }
          }
        }
        if (slot >= 0) {
          const G* row = values + int64_t(slot) * a.dim + col;
          if constexpr (kGradVector) {
            load4(row, g);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) g[i] = load1(row + i);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) g[i] = clipped(g[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = element(o + i);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) update(p[i], g[i], m[i], v[i]);
      store4(a.exp_avg + e0 + o, m);
      store4(a.exp_avg_sq + e0 + o, v);
      store4(param + e0 + o, p);
    }
  };
  if constexpr (kVector) {
    if (mostly_quiet)
      sweep(std::true_type{});
    else
      sweep(std::false_type{});
  }
  for (int o = body + threadIdx.x; o < len; o += ADAM_THREADS) {
    const int64_t e = e0 + o;
    float p1 = load1(param + e), m1 = a.exp_avg[e], v1 = a.exp_avg_sq[e];
    update(p1, element(o), m1, v1);
    a.exp_avg[e] = m1;
    a.exp_avg_sq[e] = v1;
    store1(param + e, p1);
  }
}

template <typename P, typename G>
int run_adamw_rows(const muon_adamw_rows_seg& sg, const AdamwRowsArgs& a, cudaStream_t stream) {
  const bool vec = ((reinterpret_cast<uintptr_t>(sg.param) | reinterpret_cast<uintptr_t>(sg.exp_avg) |
                     reinterpret_cast<uintptr_t>(sg.exp_avg_sq)) & 15u) == 0;
  const bool grad_vec = vec && sg.dim % ADAM_VEC == 0 && (reinterpret_cast<uintptr_t>(sg.values) & 15u) == 0;
  const int64_t blocks = (a.numel + ROWS_CHUNK - 1) / ROWS_CHUNK;
  if (blocks > 0x7fffffffLL) return set_error(MUON_ERR_ARG, "too many AdamW chunks");
  const size_t smem = sizeof(int32_t) * size_t(ROWS_CHUNK / sg.dim + 2);
  P* p = static_cast<P*>(sg.param);
  const G* g = static_cast<const G*>(sg.values);
  if (grad_vec)
    adamw_rows_kernel<P, G, true, true><<<unsigned(blocks), ADAM_THREADS, smem, stream>>>(p, g, a);
  else if (vec)
    adamw_rows_kernel<P, G, true, false><<<unsigned(blocks), ADAM_THREADS, smem, stream>>>(p, g, a);
  else
    adamw_rows_kernel<P, G, false, false><<<unsigned(blocks), ADAM_THREADS, smem, stream>>>(p, g, a);
  return check_cuda(cudaGetLastError(), "adamw rows launch");
}

int launch_adamw_rows(const muon_adamw_rows_seg* seg, double beta1, double beta2, float eps, float wd_factor,
                      const float* grad_scale, cudaStream_t stream) {
  if (!seg) return set_error(MUON_ERR_ARG, "null AdamW row segment");
  const muon_adamw_rows_seg& sg = *seg;
  if (sg.rows < 0 || sg.dim < 0 || sg.cap < 0 || sg.cap > 0x7fffffffLL || sg.dim > 0x7fff0000LL ||
      (sg.dim > 0 && (sg.rows > (int64_t(1) << 43) / sg.dim || sg.cap > (int64_t(1) << 58) / sg.dim)))
    return set_error(MUON_ERR_ARG, "AdamW row sizes out of range");
  if ((sg.param_dtype != MUON_BF16 && sg.param_dtype != MUON_F32) ||
      (sg.grad_dtype != MUON_BF16 && sg.grad_dtype != MUON_F32))
    return set_error(MUON_ERR_ARG, "AdamW row dtypes must be MUON_BF16 or MUON_F32");
  if (sg.rows == 0 || sg.dim == 0) return MUON_OK;
  if (!sg.param || !sg.exp_avg || !sg.exp_avg_sq || (sg.cap > 0 && (!sg.ids || !sg.values)))
    return set_error(MUON_ERR_ARG, "null AdamW row pointer");
  if (misaligned(sg.param, sg.param_dtype == MUON_BF16 ? 2 : 4) || misaligned(sg.exp_avg, 4) ||
      misaligned(sg.exp_avg_sq, 4) || misaligned(sg.ids, 8) || misaligned(sg.count, 8) ||
      misaligned(sg.values, sg.grad_dtype == MUON_BF16 ? 2 : 4) || misaligned(grad_scale, 4))
    return set_error(MUON_ERR_ARG, "AdamW row pointer not aligned to its dtype");
  // Blocks read and write in no fixed order: what one writes nothing else may touch.
  struct Span {
    const void* at;
    int64_t bytes;
  };
  const int64_t numel = sg.rows * sg.dim, param_size = sg.param_dtype == MUON_BF16 ? 2 : 4;
  const Span spans[] = {{sg.param, numel * param_size},
                        {sg.exp_avg, numel * 4},
                        {sg.exp_avg_sq, numel * 4},
                        {sg.ids, sg.cap * 8},
                        {sg.values, sg.cap * sg.dim * (sg.grad_dtype == MUON_BF16 ? 2 : 4)},
                        {sg.count, sg.count ? 8 : 0},
                        {grad_scale, grad_scale ? 4 : 0}};
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 7; ++j) {
      const uintptr_t x = reinterpret_cast<uintptr_t>(spans[i].at), y = reinterpret_cast<uintptr_t>(spans[j].at);
      if (spans[j].bytes > 0 && x < y + spans[j].bytes && y < x + spans[i].bytes)
        return set_error(MUON_ERR_ARG, "AdamW row buffers share memory");
    }
  AdamwRowsArgs a{};
  a.exp_avg = sg.exp_avg;
  a.exp_avg_sq = sg.exp_avg_sq;
  a.ids = sg.ids;
  a.count = sg.count;
  a.rows = sg.rows;
  a.dim = sg.dim;
  a.cap = sg.cap;
  a.numel = numel;
  a.beta1w = static_cast<float>(1.0 - beta1);
  a.beta2 = static_cast<float>(beta2);
  a.one_minus_beta2 = static_cast<float>(1.0 - beta2);
  a.eps = eps;
  a.wd_factor = wd_factor;
  a.neg_step = -sg.step_size;
  a.bc2_sqrt = sg.bc2_sqrt;
  a.grad_scale = grad_scale;
  a.quiet = eps >= 0x1p-30f && sg.bc2_sqrt > 0.f && std::fabs(sg.step_size) <= 0x1p6f;
  using bf = __nv_bfloat16;
  const bool pb = sg.param_dtype == MUON_BF16, gb = sg.grad_dtype == MUON_BF16;
  if (pb && gb) return run_adamw_rows<bf, bf>(sg, a, stream);
  if (pb) return run_adamw_rows<bf, float>(sg, a, stream);
  if (gb) return run_adamw_rows<float, bf>(sg, a, stream);
  return run_adamw_rows<float, float>(sg, a, stream);
}

int launch_adamw(const muon_adamw_seg* segs_dev, int n_segs, int64_t total_chunks, double beta1, double beta2,
                 float eps, float wd_factor, const float* grad_scale, cudaStream_t stream) {
  if (n_segs <= 0 || total_chunks <= 0) return MUON_OK;
  if (!segs_dev) return set_error(MUON_ERR_ARG, "null AdamW segment table");
  if (total_chunks > 0x7fffffffLL) return set_error(MUON_ERR_ARG, "too many AdamW chunks");
  // (1 - beta1) and (1 - beta2) are formed in double by the reference's
  // Python code and rounded to float when applied.
  const float beta1w = static_cast<float>(1.0 - beta1);
  const float omb2 = static_cast<float>(1.0 - beta2);
  adamw_kernel<<<static_cast<unsigned>(total_chunks), ADAM_THREADS, 0, stream>>>(segs_dev, n_segs, beta1w,
                                                                                 static_cast<float>(beta2), omb2, eps, wd_factor,
                                                                                 grad_scale);
  if (check_cuda(cudaGetLastError(), "adamw launch")) return MUON_ERR_CUDA;
  return MUON_OK;
}

}  // namespace muon
