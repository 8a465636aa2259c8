// The int8 KV cache's layout, shared by its own kernels and the attention
// that reads it (kv8.hip explains the choice).
#pragma once

#include "internal.h"

namespace scry {

struct Kv8Batch {  // passed to kernels by value: same n_kv and hd, own sizes
    int8_t *k[PF_MAX_SEQS], *v[PF_MAX_SEQS];
    float *ks[PF_MAX_SEQS], *vs[PF_MAX_SEQS];
    int rows_p[PF_MAX_SEQS];
    int n_kv, hd, hdp;
};

// Checks n_seq handles of one shape, each with room for rows [0, end[s]), and
// fills b; `distinct`: no handle twice (they are written).
int kv8_batch(const char *what, const scry_kv8 *caches, int n_seq, const DraftBatch &d, int rows, bool distinct,
              Kv8Batch *b);

namespace dev {
// byte of row r (of 64) inside its 64-byte group of one dimension
__device__ __forceinline__ int kv8_perm(int r) { return ((r >> 2) & 3) * 16 + (r >> 4) * 4 + (r & 3); }
__device__ __forceinline__ size_t kv8_k_at(int rows_p, int hdp, int g, int r) { return ((size_t)g * rows_p + r) * hdp; }
// the 64-byte group of dimension d that holds row r
__device__ __forceinline__ size_t kv8_v_at(int rows_p, int hdp, int g, int r, int d) {
    return (((size_t)g * rows_p + (r & ~63)) * hdp) + (size_t)d * 64;
}
}  // namespace dev
}  // namespace scry
