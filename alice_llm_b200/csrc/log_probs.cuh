// What rows of logits say about given tokens (csrc/log_probs.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace alice {

constexpr uint32_t LOGP_MAX_TOP = 32;

struct LogProbArgs {
    const float* x;              // [rows] of vocab logits, ld apart
    size_t ld;
    uint32_t rows, vocab;
    const uint32_t* target;      // [rows], or null
    float *lp, *entropy;         // [rows] each, or null
    uint32_t* rank;              // [rows], or null
    uint32_t top;                // alternatives a row, 0 .. LOGP_MAX_TOP
    uint32_t* top_ids;           // [rows][top]
    float* top_lp;               // [rows][top]
};

cudaError_t launch_log_probs(const LogProbArgs& a, int num_sms, cudaStream_t st, bool pdl);

}  // namespace alice
