// The tensor-core pass of linear attention: tensor maps, the parts of inputs that are not bf16 rows already, and the launches for bf16.
#include "linear_attention_mma.cuh"

namespace
{

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder()
{
    static const EncodeTiled found = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult result;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &result) != cudaSuccess ||
            result != cudaDriverEntryPointSuccess)
        {
            cudaGetLastError();
            return static_cast<EncodeTiled>(nullptr);
        }
        return reinterpret_cast<EncodeTiled>(fn);
    }();
    return found;
}

// A distance of one entry of a dimension that has only one entry is never used: any valid one will do.
bool stride_fits(int64_t stride, int64_t entries) { return entries <= 1 || (stride * 2 % 16 == 0 && stride > 0 && stride * 2 < (int64_t(1) << 40)); }

int64_t heads_of(const AttentionArgs &a, const TokenRows &r) { return a.heads / r.group; }

bool rows_fit(const AttentionArgs &a, const TokenRows &r)
{
    return aligned16(r.data) && stride_fits(r.head, heads_of(a, r)) && stride_fits(r.token, a.tokens) &&
           (a.offsets != nullptr || stride_fits(r.sequence, a.sequences));
}

bool make_map(CUtensorMap *map, const AttentionArgs &a, const TokenRows &r, int columns, int parts)
{
    const bool packed = a.offsets != nullptr;
    const int64_t heads = heads_of(a, r), sequences = (packed ? 1 : a.sequences) * parts;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(a.tokens),
                                static_cast<cuuint64_t>(sequences)};
    const cuuint64_t strides[3] = {heads > 1 ? static_cast<cuuint64_t>(r.head) * 2 : 256, a.tokens > 1 ? static_cast<cuuint64_t>(r.token) * 2 : 256,
                                   sequences > 1 ? static_cast<cuuint64_t>(packed ? r.token * a.tokens : r.sequence) * 2 : 256};
    const cuuint32_t box[4] = {kBoxColumns, 1, kChunk, 1}, ones[4] = {1, 1, 1, 1};
    return encoder()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, r.data, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The bf16 parts of an array, plane by plane: planes[part][sequence][token][head][columns], columns filled up to a multiple of eight
// with zeros so that tiled copies can read them.  One CTA per row (all heads of a token).
struct SplitArgs
{
    TokenRows from[4];
    __nv_bfloat16 *to[4];
    int32_t columns[4], heads[4];
    const int64_t *offsets;
    int64_t sequences, tokens;
};

template <class T, int IN>
__global__ void __launch_bounds__(256) attention_split_kernel(const __grid_constant__ SplitArgs a)
{
    const int array = blockIdx.y, columns = a.columns[array], filled = (columns + 7) / 8 * 8, heads = a.heads[array], half = filled / 2;
    const TokenRows &r = a.from[array];
    const int64_t rows = a.offsets == nullptr ? a.sequences * a.tokens : a.tokens;
    int64_t begin = 0, end = rows;
    if (a.offsets != nullptr)
    {
        // rows that no sequence owns are not read
        begin = min(max(a.offsets[0], int64_t(0)), rows);
        end = min(max(a.offsets[a.sequences], int64_t(0)), rows);
    }
    const int64_t plane = rows * heads * half;
    for (int64_t row = begin + blockIdx.x; row < end; row += gridDim.x)
    {
        const int64_t n = a.offsets == nullptr ? row / a.tokens : 0, t = a.offsets == nullptr ? row - n * a.tokens : row;
        const T *from = static_cast<const T *>(r.data) + n * r.sequence + t * r.token;
        uint32_t *to = reinterpret_cast<uint32_t *>(a.to[array]) + row * heads * half;
        for (int i = threadIdx.x; i < heads * half; i += 256)
        {
            const int h = i / half, c = (i - h * half) * 2;
            const T *x = from + h * r.head + c;
            float y[2];
            uint32_t part[IN];
#pragma unroll
            for (int e = 0; e < 2; ++e) y[e] = c + e < columns ? static_cast<float>(widen(x[e])) : 0.0f;
#pragma unroll
            for (int k = 0; k < IN; ++k)
            {
                part[k] = pack_bf16(two(y[0], y[1]));
                const float first = __uint_as_float(part[k] << 16), second = __uint_as_float(part[k] & 0xffff0000u);
                // infinities and NaN are the first part's alone
                y[0] = isfinite(first) ? y[0] - first : 0.0f;
                y[1] = isfinite(second) ? y[1] - second : 0.0f;
                to[k * plane + i] = part[k];
            }
        }
    }
}

}

namespace acro_b200_detail
{

int attention_mma_bf16(const AttentionArgs &a, const void *maps, int q, int v, bool states_only, cudaStream_t stream)
{
    return launch_parts<1, __nv_bfloat16>(a, *static_cast<const Maps *>(maps), q, v, states_only, stream);
}

// Sizes that the pass takes: at most 128 columns, 31-bit numbers of tokens and sequences.
bool attention_mma_sizes(const AttentionArgs &a)
{
    if (a.tokens < 1 || a.tokens > INT32_MAX - 2 * kChunk || a.sequences > INT32_MAX / 4 || encoder() == nullptr) return false;
    for (int i = 0; i < a.passes; ++i)
    {
        const AttentionPass &p = a.pass[i];
        if (p.dq > 128 || p.dv > 128 || p.out.token < 0 || p.out.token > (1 << 29)) return false;
    }
    return true;
}

// bf16 rows that tiled copies can read as they are: 16-byte boundaries and strides.
bool attention_mma_direct(const AttentionArgs &a)
{
    for (int i = 0; i < a.passes; ++i)
    {
        const AttentionPass &p = a.pass[i];
        if (!rows_fit(a, p.q) || !rows_fit(a, p.k) || !rows_fit(a, p.v)) return false;
    }
    return true;
}

int attention_parts(int type) { return type == ACRO_B200_F32 ? 3 : type == ACRO_B200_F16 ? 2 : 1; }

size_t attention_planes_bytes(int type, int64_t rows, int heads, int columns)
{
    return (static_cast<size_t>(attention_parts(type)) * rows * heads * ((columns + 7) / 8 * 8) * 2 + 255) / 256 * 256;
}

int attention_split(AttentionArgs &a, int type, const TokenRows *arrays, const int *columns, int count, void *planes, cudaStream_t stream)
{
    const bool packed = a.offsets != nullptr;
    const int64_t rows = packed ? a.tokens : a.sequences * a.tokens;
    SplitArgs s = {};
    s.offsets = a.offsets;
    s.sequences = a.sequences;
    s.tokens = a.tokens;
    TokenRows plane[4];
    unsigned char *at = static_cast<unsigned char *>(planes);
    for (int i = 0; i < count; ++i)
    {
        const int heads = static_cast<int>(heads_of(a, arrays[i])), filled = (columns[i] + 7) / 8 * 8;
        s.from[i] = arrays[i];
        s.to[i] = reinterpret_cast<__nv_bfloat16 *>(at);
        s.columns[i] = columns[i];
        s.heads[i] = heads;
        plane[i] = {at, static_cast<int64_t>(heads) * filled * a.tokens, static_cast<int64_t>(heads) * filled, filled, arrays[i].group};
        at += attention_planes_bytes(type, rows, heads, columns[i]);
    }
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(rows, 148 * 32)), count);
    if (type == ACRO_B200_F32) attention_split_kernel<float, 3><<<grid, 256, 0, stream>>>(s);
    else if (type == ACRO_B200_F16) attention_split_kernel<__half, 2><<<grid, 256, 0, stream>>>(s);
    else attention_split_kernel<__nv_bfloat16, 1><<<grid, 256, 0, stream>>>(s);
    for (int i = 0; i < a.passes; ++i)
    {
        AttentionPass &p = a.pass[i];
        for (TokenRows *r : {&p.q, &p.k, &p.v})
            for (int k = 0; k < count; ++k)
                if (r->data == arrays[k].data && r->sequence == arrays[k].sequence && r->token == arrays[k].token && r->head == arrays[k].head &&
                    r->group == arrays[k].group && (r == &p.v ? p.dv : p.dq) == columns[k])
                {
                    *r = plane[k];
                    break;
                }
    }
    return launch_status("acro_b200_linear_attention");
}

int attention_mma_launch(const AttentionArgs &a, int type, bool states_only, cudaStream_t stream)
{
    Maps maps = {};
    int q = 1, v = 1;
    const int parts = attention_parts(type);
    maps.sequences = a.offsets != nullptr ? 1 : static_cast<int32_t>(a.sequences);
    for (int i = 0; i < a.passes; ++i)
    {
        const AttentionPass &p = a.pass[i];
        q = std::max(q, (p.dq + 63) / 64);
        v = std::max(v, (p.dv + 63) / 64);
        if (!make_map(&maps.q[i], a, p.q, p.dq, parts) || !make_map(&maps.k[i], a, p.k, p.dq, parts) || !make_map(&maps.v[i], a, p.v, p.dv, parts))
            return fail_cuda(cudaErrorInvalidValue, "acro_b200_linear_attention (tensor map)");
    }
    if (a.items * a.heads > INT32_MAX) return fail_unsupported("acro_b200_linear_attention: more than 2^31 segments x heads");
    if (parts == 3) return attention_mma_f32(a, &maps, q, v, states_only, stream);
    return parts == 2 ? attention_mma_f16(a, &maps, q, v, states_only, stream) : attention_mma_bf16(a, &maps, q, v, states_only, stream);
}

}
