/*
 * attn_view.cuh — what the attention kernels are given (include/backend_cuda.h, ApusCudaAttn).
 */
#pragma once
#include <stdint.h>

namespace apus {

struct AttnView {
    const uint16_t *q, *gate;
    uint16_t *out;
    float *lse;
    long q_stride, gate_stride, out_stride;
    int rows, heads, group;
    float scale;
};

}  // namespace apus
