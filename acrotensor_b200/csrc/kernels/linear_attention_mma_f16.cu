// The tensor-core pass of linear attention for fp16: inputs of two bf16 parts.
#include "linear_attention_mma.cuh"

namespace acro_b200_detail
{

int attention_mma_f16(const AttentionArgs &a, const void *maps, int q, int v, bool states_only, cudaStream_t stream)
{
    return launch_parts<2, __half>(a, *static_cast<const Maps *>(maps), q, v, states_only, stream);
}

}
