// What the masked attention's host and device sides share (masked_attention.cu).
#pragma once
#include <cuda_runtime.h>

#include "../../include/monofab.h"

namespace mf {

using MaskedAttnParams = monofab_masked_attention_args;

}  // namespace mf
