// attn_prefill.hpp — causal attention over packed short prompts on F32 MFMA
// (attn_prefill.hip), used by the packed entry points.
#pragma once

#include <hip/hip_runtime.h>

#include "batch.hpp"
#include "ikv_common.hpp"

namespace ikv {

// Operands as for attn_bf16x3_packed (attn_bf16x3.hpp). -ENOTSUP for what
// it does not take, or where the other kernels are expected to be faster.
int attn_prefill_packed(const float *q, const float *k, const float *v, const Pages *pages, float *out,
                        int n_head, int n_head_kv, int head_dim, const PackedSeqs &seqs, float scale,
                        hipStream_t s);

}  // namespace ikv
