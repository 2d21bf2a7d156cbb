// Launchers of the decoder operators (include/lunara_b200_decoder.h), behind
// the argument checks of decoder_abi.cu.
#pragma once

#include <cuda_runtime.h>

#include "../../include/lunara_b200_decoder.h"

namespace lunara {

cudaError_t launch_rotary(const lunarad_rotary_args& a, cudaStream_t stream);
cudaError_t launch_qk_norm_rotary(const lunarad_qk_norm_rotary_args& a, cudaStream_t stream);
cudaError_t launch_kv_append(const lunarad_kv_append_args& a, cudaStream_t stream);
cudaError_t launch_kv_read(const lunarad_kv_read_args& a, cudaStream_t stream);
int64_t paged_attention_workspace(const lunarad_paged_attention_args& a, int sms);
cudaError_t launch_paged_attention(const lunarad_paged_attention_args& a, void* workspace, cudaStream_t stream);

}  // namespace lunara
