// The tensor-core pass of linear attention for fp32: inputs of three bf16 parts.
#include "linear_attention_mma.cuh"

namespace acro_b200_detail
{

int attention_mma_f32(const AttentionArgs &a, const void *maps, int q, int v, bool states_only, cudaStream_t stream)
{
    return launch_parts<3, float>(a, *static_cast<const Maps *>(maps), q, v, states_only, stream);
}

}
