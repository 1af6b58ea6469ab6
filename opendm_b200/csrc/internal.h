// Internal (C++) interface between the C-ABI layer and the kernel files.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "opendm_muon.h"

namespace muon {

// Records a failure for muon_last_error() and returns `code`.
int set_error(int code, const std::string& msg);
// Whether a pointer's elements of `bytes` would straddle their natural boundary, which faults.
inline bool misaligned(const void* p, unsigned bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }
int check_cuda(cudaError_t e, const char* what);

int launch_momentum(const muon_momentum_seg* segs_dev, int n_segs, int64_t total_chunks,
                    int grad_dtype, int dir_dtype, float momentum, int nesterov, float eps,
                    float* partials_dev, float* scales_dev, const float* grad_scale, cudaStream_t stream);
int64_t momentum_chunks(int64_t rows, int64_t cols);
int launch_momentum_single_noalloc(const void* grad, float* exp_avg, void* direction, int64_t rows, int64_t cols,
                                   int64_t ld, int grad_dtype, int dir_dtype, float momentum, int nesterov,
                                   float eps, float* scale_out, cudaStream_t stream);

int launch_adamw(const muon_adamw_seg* segs_dev, int n_segs, int64_t total_chunks, double beta1,
                 double beta2, float eps, float wd_factor, const float* grad_scale, cudaStream_t stream);
int64_t norm_chunks(int64_t numel);
int launch_clip_grad_norm(const muon_norm_seg* segs_dev, int n_segs, int64_t total_chunks, float max_norm,
                          float* partials_dev, float* out_dev, cudaStream_t stream);
int64_t adamw_chunks(int64_t numel);

int ns_plan_create(const muon_ns_class* classes, int n_classes, int op_dtype, int steps,
                   muon_ns_plan** plan_out);
int ns_plan_run(const muon_ns_plan* plan, int* err_dev, cudaStream_t stream);
int launch_apply_update(const muon_update_seg* segs_dev, int n_segs, int64_t total_chunks, float wd_factor,
                        cudaStream_t stream);
void ns_plan_destroy(muon_ns_plan* plan);
int ns_plan_launches(const muon_ns_plan* plan);
int ns_plan_set_sm_limit(muon_ns_plan* plan, int sms);
int64_t ns_class_workspace_bytes(int32_t rows, int32_t cols, int32_t count, int op_dtype, int algo);
int ns_choose_algo(int32_t rows, int32_t cols, int op_dtype, int steps);
int ns_gram_segment(int op_dtype);
int ns_class_layout(muon_ns_class* cls, void* base, int op_dtype);
float ns_operand_scale(int32_t rows, int32_t cols, int iteration, int op_dtype);

int launch_flags_set(const muon_flag_list* list, uint32_t value, cudaStream_t stream);
int launch_flags_wait(const muon_flag_list* list, uint32_t value, int64_t timeout_us, int* err_dev,
                      cudaStream_t stream);

int launch_momentum_f16(const muon_momentum_f16_seg* segs_dev, int n_segs, int64_t total_chunks, int grad_dtype,
                        float momentum, int nesterov, float eps, float* partials_dev, float* pscale_dev,
                        float* scales_dev, int* redo_dev, const float* grad_scale, cudaStream_t stream);

// Launches `kernel` so that it may start while the kernel before it on the
// stream (one of this library that calls allow_next()) drains; it has to call
// wait_previous() before it touches memory. Its pointers are never
// __restrict__: const ones would promise that nothing writes their memory
// while the kernel runs, which its predecessor does until that wait, and so
// let loads use the non-coherent path or move above it.
template <typename... Params, typename... Args>
int launch_overlapped(const char* what, void (*kernel)(Params...), unsigned grid, unsigned block, cudaStream_t stream,
                      Args... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, Params(args)...), what);
}

int launch_adamw_rows(const muon_adamw_rows_seg* seg, double beta1, double beta2, float eps, float wd_factor,
                      const float* grad_scale, cudaStream_t stream);

int launch_embedding(const void* weight, int weight_dtype, int64_t rows, int64_t dim, int64_t ld, const void* ids,
                     int ids_dtype, int64_t tokens, float scale, void* out, int out_dtype, int* err,
                     cudaStream_t stream);
int64_t embedding_grad_workspace_bytes(int64_t tokens, int64_t rows, int64_t dim);
int launch_embedding_grad(const void* grad, int grad_dtype, const void* ids, int ids_dtype, int64_t tokens,
                          int64_t rows, int64_t dim, int64_t padding_idx, float scale, void* out, int out_dtype,
                          int64_t* out_ids, int64_t* count, void* workspace, int64_t workspace_bytes, int* err,
                          cudaStream_t stream);

int64_t clip_workspace_bytes(int64_t n_segs);
int launch_total_norm(const muon_clip_seg* segs, int64_t n_segs, int norm_kind, void* workspace, float* total,
                      cudaStream_t stream);
int launch_clip_grads(const muon_clip_seg* segs, int64_t n_segs, int norm_kind, float max_norm, void* workspace,
                      float* total, cudaStream_t stream);
int launch_scale_grads(const muon_clip_seg* segs, int64_t n_segs, float max_norm, const float* total,
                       cudaStream_t stream);
}  // namespace muon
