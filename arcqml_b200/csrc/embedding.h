// embedding.h — rows of a table looked up by index, and that lookup's gradient (embedding.cu).
#pragma once

#include "../../include/arcqml_runtime_v2.h"
#include "rt_internal.h"

namespace arcqml {

// Doubles of device scratch (0: none).
size_t embedding_lookup_workspace(const ArcqmlRows &table, size_t count, const ArcqmlEmbeddingOptions &o);
size_t embedding_gradient_workspace(const ArcqmlRows &gradient, uint64_t rows,
                                    const ArcqmlEmbeddingOptions &o);
// out[i] <- scale table[indices[i]] (over the row's norm).
void embedding_lookup_device(const ArcqmlRows &table, const void *indices, size_t count,
                             const ArcqmlEmbeddingOptions &o, const ArcqmlRows &out, double *ws,
                             size_t ws_len, cudaStream_t s);
// out[v] <- scale times the sum of the gradient's rows whose index is v (through the row's norm).
void embedding_gradient_device(const ArcqmlRows &gradient, const void *indices,
                               const ArcqmlEmbeddingOptions &o, const ArcqmlRows *table,
                               const ArcqmlRows &out, double *ws, size_t ws_len, cudaStream_t s);

}  // namespace arcqml
