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
// with zeros so that tiled copies can read them.  A CTA takes a few rows (all heads of a token), a thread four columns at a time.
struct SplitArgs
{
    TokenRows from[4];
    __nv_bfloat16 *to[4];
    int32_t columns[4], heads[4], packs[4];     // packs: four columns can be read at once
    const int64_t *offsets;
    int64_t sequences, tokens;
};

// Rows that a CTA of the split kernel takes at once, `each` quads of columns a row.
__host__ __device__ __forceinline__ int split_at_once(int each) { return each >= 1024 ? 1 : 1024 / each; }

// Infinities and NaN among two values as bf16, with zeros in their place.
__device__ __forceinline__ uint32_t take_odd(Two &x)
{
    const bool first = !isfinite(first_of(x)), second = !isfinite(second_of(x));
    const uint32_t all = pack_bf16(x);
    x = two(first ? 0.0f : first_of(x), second ? 0.0f : second_of(x));
    return (first ? all & 0xffffu : 0u) | (second ? all & 0xffff0000u : 0u);
}

// Six CTAs an SM: with the 62 registers that fp32 takes otherwise, and four CTAs, 4 x 1024 rows of 12 heads of 64 took 27 us instead of 24.5.
template <class T, int IN>
__global__ void __launch_bounds__(256, 6) attention_split_kernel(const __grid_constant__ SplitArgs a)
{
    const int array = blockIdx.y, columns = a.columns[array], heads = a.heads[array], quads = (columns + 7) / 8 * 2, each = heads * quads;
    const TokenRows &r = a.from[array];
    const bool packs = a.packs[array] != 0;
    const int64_t rows = a.offsets == nullptr ? a.sequences * a.tokens : a.tokens;
    int64_t begin = 0, end = rows;
    if (a.offsets != nullptr)
    {
        // rows that no sequence owns are not read (where sequences are skipped, all rows are)
        const int64_t from = a.offsets[0], to = a.offsets[a.sequences];
        if (offsets_ascend(a.offsets, a.sequences, rows))
        {
            begin = from;
            end = to;
        }
    }
    const int some = split_at_once(each);
    const int64_t plane = rows * each;
    for (int64_t first = begin + static_cast<int64_t>(blockIdx.x) * some; first < end; first += static_cast<int64_t>(gridDim.x) * some)
    {
        const int count = static_cast<int>(min(static_cast<int64_t>(some), end - first)) * each;
        uint2 *to = reinterpret_cast<uint2 *>(a.to[array]) + first * each;
#pragma unroll 2
        for (int i = threadIdx.x; i < count; i += 256)
        {
            const int own = i / each, rest = i - own * each, h = rest / quads, c = (rest - h * quads) * 4;
            const int64_t row = first + own, n = a.offsets == nullptr ? row / a.tokens : 0, t = row - n * a.tokens;
            const T *x = static_cast<const T *>(r.data) + n * r.sequence + t * r.token + h * r.head + c;
            Two y[2];
            if (packs && c < columns)
            {
                const Pack<T, 4> p = load_pack<T, 4>(x);
                y[0] = two(widen(p.x[0]), widen(p.x[1]));
                y[1] = two(widen(p.x[2]), widen(p.x[3]));
            }
            else
            {
                float z[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) z[e] = c + e < columns ? static_cast<float>(widen(x[e])) : 0.0f;
                y[0] = two(z[0], z[1]);
                y[1] = two(z[2], z[3]);
            }
            // infinities and NaN are the first part's alone; finite values have finite parts, above the largest bf16 too
            // (no branch: it would keep the next values' loads behind it)
            const uint2 odd = make_uint2(take_odd(y[0]), take_odd(y[1]));
#pragma unroll
            for (int k = 0; k < IN; ++k)
            {
                uint2 part = make_uint2(take_part(y[0]), take_part(y[1]));
                if (k == 0) part = make_uint2(part.x | odd.x, part.y | odd.y);
                to[k * plane + i] = part;
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
    int some = 1024;
    unsigned char *at = static_cast<unsigned char *>(planes);
    for (int i = 0; i < count; ++i)
    {
        const int heads = static_cast<int>(heads_of(a, arrays[i])), filled = (columns[i] + 7) / 8 * 8;
        s.from[i] = arrays[i];
        s.to[i] = reinterpret_cast<__nv_bfloat16 *>(at);
        s.columns[i] = columns[i];
        const int64_t pack = 4 * (type == ACRO_B200_F32 ? 4 : 2);
        s.packs[i] = columns[i] % 4 == 0 && reinterpret_cast<uintptr_t>(arrays[i].data) % pack == 0 && arrays[i].sequence % 4 == 0 && arrays[i].token % 4 == 0 &&
                     arrays[i].head % 4 == 0;
        s.heads[i] = heads;
        some = std::min(some, split_at_once(heads * filled / 4));
        plane[i] = {at, static_cast<int64_t>(heads) * filled * a.tokens, static_cast<int64_t>(heads) * filled, filled, arrays[i].group};
        at += attention_planes_bytes(type, rows, heads, columns[i]);
    }
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((rows + some - 1) / some, 148 * 8)), count);
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
