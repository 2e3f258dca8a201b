// muon.h — matrices orthogonalised by Newton-Schulz products, and the momentum step with them (muon.cu).
#pragma once

#include "../../include/arcqml_runtime_v2.h"
#include "rt_internal.h"

namespace arcqml {

// Doubles of device scratch for a list.
size_t orthogonalize_workspace(const ArcqmlMatrix *list, size_t count);
void orthogonalize_device(const ArcqmlMatrix *in, const ArcqmlMatrix *out, size_t count, int steps,
                          double eps, double *ws, size_t ws_len, cudaStream_t s);
void muon_step_device(const ArcqmlMatrix *params, const ArcqmlMatrix *grads, const ArcqmlMatrix *momenta,
                      size_t count, const ArcqmlMuonOptions &o, double *ws, size_t ws_len, cudaStream_t s);

}  // namespace arcqml
