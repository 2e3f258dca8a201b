// optim.h — training over many device tensors (optim.cu): global gradient norm, clipping, Adam.
#pragma once

#include "../../include/arcqml_runtime_v2.h"
#include "rt_internal.h"

namespace arcqml {

// Doubles of device scratch for a list of gradients, and for a list of parameters (0: a short list,
// one launch).
size_t gradient_workspace(const ArcqmlTensor *list, size_t count);
size_t adam_workspace(const ArcqmlTensor *list, size_t count);
// *norm (device) <- 2-norm over all elements of all tensors.
void gradient_norm_device(const ArcqmlTensor *grads, size_t count, double *norm, double *ws,
                          size_t ws_len, cudaStream_t s);
// grads <- min(1, max_norm / (n + 1e-6)) grads, n = *given (device) or the list's norm.
void clip_gradients_device(const ArcqmlTensor *grads, size_t count, double max_norm,
                           const double *given, double *norm, double *ws, size_t ws_len,
                           cudaStream_t s);
// One Adam step with the clip factor folded in; *step (device) is advanced.
void adam_step_device(const ArcqmlTensor *params, const ArcqmlTensor *grads,
                      const ArcqmlTensor *m, const ArcqmlTensor *v, const ArcqmlTensor *copies,
                      size_t count, int64_t *step, const ArcqmlAdamOptions &o,
                      const double *given, double *norm, double *ws, size_t ws_len,
                      cudaStream_t s);

}  // namespace arcqml
