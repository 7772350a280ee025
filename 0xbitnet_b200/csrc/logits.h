// logits.h — penalties, biases and grammar masks on rows of logits (logits.cu).
#pragma once

#include <cstddef>
#include <cstdint>

#include <cuda_runtime.h>

#include "../../include/obn.h"

namespace obn {

// obn_logits_process (include/obn.h) after its checks; token may be null.
cudaError_t launch_logits_process(const float* logits, int rows, int vocab,
                                  const obn_logit_rules& rules, float* out, int32_t* token,
                                  cudaStream_t s);

}  // namespace obn
