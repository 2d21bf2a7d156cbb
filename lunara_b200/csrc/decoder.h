// Launchers of the decoder operators (include/lunara_b200_decoder.h), behind
// the argument checks of decoder_abi.cu.
#pragma once

#include <cuda_runtime.h>

#include "../../include/lunara_b200_decoder.h"

namespace lunara {

cudaError_t launch_rotary(const lunarad_rotary_args& a, cudaStream_t stream);
cudaError_t launch_qk_norm_rotary(const lunarad_qk_norm_rotary_args& a, cudaStream_t stream);
// zero_rest: LUNARAD_ZERO_REST, which the arguments' dtype no longer holds here.
cudaError_t launch_kv_append(const lunarad_kv_append_args& a, bool zero_rest, cudaStream_t stream);
cudaError_t launch_kv_read(const lunarad_kv_read_args& a, bool zero_rest, cudaStream_t stream);
int64_t paged_attention_workspace(const lunarad_paged_attention_args& a, int sms);
cudaError_t launch_paged_attention(const lunarad_paged_attention_args& a, bool zero_rest, void* workspace, cudaStream_t stream);

}  // namespace lunara
