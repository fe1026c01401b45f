// Windowed attention on the tensor cores (attn_tensor.cu): bf16.
#pragma once
#include "attn_common.cuh"

namespace ncn {

bool attn_tensor_covers(const AttnParams& p, int dtype);
cudaError_t launch_attn_tensor_fwd(const AttnParams& p, cudaStream_t st);
cudaError_t launch_attn_tensor_bwd(const AttnParams& p, cudaStream_t st);

}  // namespace ncn
