// Linear attention with a decay for each head: entry points, the kernels for every type and head size, the step for single
// tokens.  linear_attention.cuh has the mathematics; linear_attention_mma.cuh the main pass on the tensor cores.
#include "linear_attention.cuh"

#include <algorithm>

using namespace acro_b200_detail;

namespace
{

constexpr int kThreads = 256;
constexpr int kMaxHead = 256;           // columns of a head
constexpr int kJoin = 8;                // segments whose states a thread of the join has in flight

// Rows of shared memory are read in 16-byte packs: an odd number of packs a row keeps 8 consecutive rows in different banks.
template <class A>
__host__ __device__ constexpr int padded(int columns)
{
    constexpr int n = 16 / sizeof(A);
    const int packs = (columns + n - 1) / n;
    return (packs | 1) * n;
}

// The pass works on CHUNK tokens at a time and SLICE columns of v (of the state) per CTA.
template <class A, int CHUNK, int SLICE>
size_t pass_smem_bytes(int dq)
{
    const int rows = (dq + 16 / sizeof(A) * 16 - 1) / (16 / sizeof(A) * 16) * (16 / sizeof(A) * 16);
    return sizeof(A) * (CHUNK * static_cast<size_t>(padded<A>(dq) + std::max(padded<A>(dq), padded<A>(CHUNK))) + CHUNK * SLICE +
                        static_cast<size_t>(rows) * SLICE + CHUNK + 1);
}

template <class A> struct alignas(16) Vec { A x[16 / sizeof(A)]; };

__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ bool not_finite(double x) { return (__double2hiint(x) & 0x7ff00000) == 0x7ff00000; }

// Rows 0 .. rows-1 of `to` (columns 0 .. width-1, a multiple of a pack of sums) from m rows of `from` with `columns` columns; zeros where
// there is nothing.  `packs`: rows start on 16-byte boundaries and columns are a multiple of a pack of elements.  Returns whether
// this thread met an infinity or NaN.
template <class T>
__device__ __forceinline__ bool stage_rows(typename Element<T>::Acc *to, int ld, int width, const T *from, int64_t stride, int rows, int m, int columns,
                                           bool packs)
{
    using A = typename Element<T>::Acc;
    constexpr int N = 16 / sizeof(A);
    const int each = width / N;
    bool odd = false;
    for (int i = threadIdx.x; i < rows * each; i += kThreads)
    {
        const int r = i / each, c = (i - r * each) * N;
        const T *at = from + r * stride + c;
        Vec<A> x;
        if (r < m && packs && c < columns)
        {
            const Pack<T, N> p = load_pack<T, N>(at);
#pragma unroll
            for (int k = 0; k < N; ++k) x.x[k] = widen(p.x[k]);
        }
        else
        {
#pragma unroll
            for (int k = 0; k < N; ++k) x.x[k] = r < m && c + k < columns ? static_cast<A>(widen(at[k])) : A(0);
        }
#pragma unroll
        for (int k = 0; k < N; ++k) odd |= not_finite(x.x[k]);
        *reinterpret_cast<Vec<A> *>(to + r * ld + c) = x;
    }
    return odd;
}

// acc[i][j] += sum_(s < n) P[ty + 16 i][s] V[s][column j of tx]; with GUARD only over the s that row ty + 16 i sees, because a product
// of a masked zero with an infinity or NaN of another token would be NaN.
template <class A, int TM, int NP, int SV, bool GUARD>
__device__ __forceinline__ void product(A (&acc)[TM][NP][16 / sizeof(A)], const A *p, int ldp, const A *v, int n, int ty, int tx, bool reverse)
{
    constexpr int VN = 16 / sizeof(A);
#pragma unroll 1
    for (int s = 0; s < n; s += VN)
    {
        Vec<A> row[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i) row[i] = *reinterpret_cast<const Vec<A> *>(p + (ty + 16 * i) * ldp + s);
#pragma unroll
        for (int k = 0; k < VN; ++k)
#pragma unroll
            for (int q = 0; q < NP; ++q)
            {
                const Vec<A> col = *reinterpret_cast<const Vec<A> *>(v + (s + k) * SV + (q * 16 + tx) * VN);
#pragma unroll
                for (int i = 0; i < TM; ++i)
                {
                    if (GUARD && (reverse ? s + k < ty + 16 * i : s + k > ty + 16 * i)) continue;
#pragma unroll
                    for (int j = 0; j < VN; ++j) acc[i][q][j] += row[i].x[k] * col.x[j];
                }
            }
    }
}

// The pass for every type and head size: sums of products in the type of sums on the ordinary cores, a chunk of Q, K and V, the scores
// and the state in shared memory, register tiles per thread (4 x 4 of a chunk of 64 tokens and 64 columns; 2 x 8 of 32 tokens and 128
// columns; in 64 bits 2 x 2).  Bound by those cores and by their reads of shared memory, not by HBM.
template <class T, int C, int SV>
__global__ void __launch_bounds__(kThreads) attention_pass_kernel(const __grid_constant__ AttentionArgs a, int slices, bool states_only)
{
    using A = typename Element<T>::Acc;
    constexpr int VN = 16 / sizeof(A), TM = C / 16, NP = SV / 16 / VN;
    const AttentionPass &p = a.pass[blockIdx.y];
    const int head = blockIdx.x % a.heads, slice = blockIdx.x / a.heads % slices;
    const int c0 = slice * SV;
    if (c0 >= p.dv) return;
    const int64_t item_index = blockIdx.x / (a.heads * slices);
    const bool reverse = p.reverse != 0;
    const SegmentItem item = find_item(a, item_index, reverse);
    if (item.sequence < 0) return;
    const bool cut = segments_of(item.sequence_end - item.sequence_begin, a.segment) > 1;
    if (states_only && (!cut || item.last)) return;

    extern __shared__ __align__(16) unsigned char smem_bytes[];
    const int ld = padded<A>(p.dq), ldp = padded<A>(C), cols = min(SV, p.dv - c0), width = (p.dq + VN - 1) / VN * VN;
    const int state_rows = (p.dq + VN * 16 - 1) / (VN * 16) * (VN * 16);
    A *sq = reinterpret_cast<A *>(smem_bytes), *sp = sq, *sk = sq + C * max(ld, ldp), *sv = sk + C * ld, *st = sv + C * SV, *power = st + state_rows * SV;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;

    const double g = decay_log<A>(a.log_decay, head);
    for (int i = threadIdx.x; i <= C; i += kThreads) power[i] = static_cast<A>(exp(g * i));

    // the state this segment starts from
    const int64_t size = static_cast<int64_t>(p.dq) * p.dv;
    const A *from = nullptr;
    int turned = 0;
    if (!states_only)
    {
        if (cut) from = static_cast<const A *>(p.segment_states) + (item.segment_state * a.heads + head) * size;
        else if (p.initial != nullptr)
        {
            from = static_cast<const A *>(p.initial) + (item.state * a.heads + head) * size;
            turned = p.turned;
        }
    }
    const int along = turned ? 1 : p.dv, across = turned ? p.dq : 1;
#pragma unroll 8
    for (int i = threadIdx.x; i < state_rows * SV; i += kThreads)
    {
        const int d = i / SV, c = i % SV;
        st[i] = from != nullptr && d < p.dq && c < cols ? from[d * along + (c0 + c) * across] : A(0);
    }
    const T *q = rows_of<const T>(p.q, a, item.sequence, head), *k = rows_of<const T>(p.k, a, item.sequence, head),
            *v = rows_of<const T>(p.v, a, item.sequence, head) + c0;
    const bool packs = p.packs != 0;
    const A scale = static_cast<A>(p.state_scale), out_scale = static_cast<A>(p.out_scale);

    const int chunks = static_cast<int>((item.end - item.begin + C - 1) / C);
    for (int index = 0; index < chunks; ++index)
    {
        const int64_t t0 = item.begin + static_cast<int64_t>(reverse ? chunks - 1 - index : index) * C;
        const int m = static_cast<int>(min(static_cast<int64_t>(C), item.end - t0));
        __syncthreads();
        // rows behind the chunk's last token and columns behind the head's last one are zeros
        if (!states_only) stage_rows<T>(sq, ld, width, q + t0 * p.q.token, p.q.token, C, m, p.dq, packs);
        stage_rows<T>(sk, ld, width, k + t0 * p.k.token, p.k.token, C, m, p.dq, packs);
        const bool odd = __syncthreads_or(stage_rows<T>(sv, SV, SV, v + t0 * p.v.token, p.v.token, C, m, cols, packs)) != 0;
        if (!states_only)
        {
            A acc[TM][TM];
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j) acc[i][j] = 0;
#pragma unroll 2
            for (int d = 0; d < p.dq; d += VN)
            {
                Vec<A> x[TM], y[TM];
#pragma unroll
                for (int i = 0; i < TM; ++i)
                {
                    x[i] = *reinterpret_cast<const Vec<A> *>(sq + (ty + 16 * i) * ld + d);
                    y[i] = *reinterpret_cast<const Vec<A> *>(sk + (tx + 16 * i) * ld + d);
                }
#pragma unroll
                for (int n = 0; n < VN; ++n)
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int j = 0; j < TM; ++j) acc[i][j] += x[i].x[n] * y[j].x[n];
            }
            A near[TM][NP][VN], far[TM][NP][VN];
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int n = 0; n < NP; ++n)
#pragma unroll
                    for (int j = 0; j < VN; ++j) near[i][n][j] = far[i][n][j] = 0;
            product<A, TM, NP, SV, false>(far, sq, ld, st, p.dq, ty, tx, reverse);
            __syncthreads();            // the scores take Q's place
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j)
                {
                    const int r = ty + 16 * i, s = tx + 16 * j, n = reverse ? s - r : r - s;
                    sp[r * ldp + s] = n < 0 ? A(0) : acc[i][j] * power[n] * scale;
                }
            __syncthreads();
            if (odd) product<A, TM, NP, SV, true>(near, sp, ldp, sv, C, ty, tx, reverse);
            else product<A, TM, NP, SV, false>(near, sp, ldp, sv, C, ty, tx, reverse);
#pragma unroll
            for (int i = 0; i < TM; ++i)
            {
                const int r = ty + 16 * i;
                if (r >= m) continue;
                const A come = power[reverse ? m - 1 - r : r + 1];
                const int64_t at = (t0 + r) * p.out.token + c0;
#pragma unroll
                for (int n = 0; n < NP; ++n)
#pragma unroll
                    for (int j = 0; j < VN; ++j)
                    {
                        const int c = (n * 16 + tx) * VN + j;
                        if (c >= cols) continue;
                        const A o = out_scale * (near[i][n][j] + come * far[i][n][j]);
                        if (p.sums) rows_of<A>(p.out, a, item.sequence, head)[at + c] = o;
                        else rows_of<T>(p.out, a, item.sequence, head)[at + c] = narrow<T>(o);
                    }
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < C * SV / VN; i += kThreads)
        {
            const int r = i / (SV / VN);
            if (r >= m) continue;
            const A w = power[reverse ? r + 1 : m - 1 - r] * scale;
            Vec<A> &x = reinterpret_cast<Vec<A> *>(sv)[i];
#pragma unroll
            for (int j = 0; j < VN; ++j) x.x[j] *= w;
        }
        __syncthreads();
        // what is left of the state after m tokens, to twice the digits: the rounding of one factor would come back in every chunk
        const double exact = exp(g * m);
        const A keep = static_cast<A>(exact), rest = static_cast<A>(exact - static_cast<double>(keep));
        for (int d = ty * VN; d < p.dq; d += 16 * VN)
        {
            A acc[VN][NP][VN];
#pragma unroll
            for (int i = 0; i < VN; ++i)
#pragma unroll
                for (int n = 0; n < NP; ++n)
#pragma unroll
                    for (int j = 0; j < VN; ++j) acc[i][n][j] = 0;
#pragma unroll 2
            for (int s = 0; s < m; ++s)
            {
                const Vec<A> x = *reinterpret_cast<const Vec<A> *>(sk + s * ld + d);
#pragma unroll
                for (int n = 0; n < NP; ++n)
                {
                    const Vec<A> y = *reinterpret_cast<const Vec<A> *>(sv + s * SV + (n * 16 + tx) * VN);
#pragma unroll
                    for (int i = 0; i < VN; ++i)
#pragma unroll
                        for (int j = 0; j < VN; ++j) acc[i][n][j] += x.x[i] * y.x[j];
                }
            }
#pragma unroll
            for (int i = 0; i < VN; ++i)
#pragma unroll
                for (int n = 0; n < NP; ++n)
                {
                    Vec<A> &s = *reinterpret_cast<Vec<A> *>(st + (d + i) * SV + (n * 16 + tx) * VN);
#pragma unroll
                    for (int j = 0; j < VN; ++j) s.x[j] = keep * s.x[j] + (rest * s.x[j] + acc[i][n][j]);
                }
        }
    }
    __syncthreads();
    A *to = nullptr;
    turned = 0;
    if (states_only) to = static_cast<A *>(p.segment_states) + (item.segment_state * a.heads + head) * size;
    else if (item.last && p.final != nullptr)
    {
        to = static_cast<A *>(p.final) + (item.state * a.heads + head) * size;
        turned = p.turned;
    }
    if (to == nullptr) return;
    for (int i = threadIdx.x; i < p.dq * SV; i += kThreads)
    {
        const int d = i / SV, c = i % SV;
        if (c < cols) to[turned ? (c0 + c) * p.dq + d : d * p.dv + c0 + c] = st[i];
    }
}

// Turns the segments' own states into the states that they start from: one thread per entry of a state, walking a sequence's
// segments in the order of time, 16 loads ahead.  Bound by the latency of offsets, powers and loads: 20 us with cold caches for 12 segments
// of 16 heads of 128 x 128 (25 MB).  Taking the powers behind the first loads did not shorten it; with the power taken in every step and
// one load at a time 144 segments took 89 us.
template <class A>
__global__ void __launch_bounds__(kThreads) attention_join_kernel(const __grid_constant__ AttentionArgs a)
{
    __shared__ double left[2];
    const AttentionPass &p = a.pass[blockIdx.z];
    const int head = blockIdx.x % a.heads;
    const int64_t n = blockIdx.x / a.heads;
    const bool reverse = p.reverse != 0;
    int64_t begin = 0, end = a.tokens;
    if (a.offsets != nullptr && !rows_of_sequence(a.offsets, n, a.tokens, INT64_MIN, begin, end)) return;
    const int64_t count = segments_of(end - begin, a.segment);
    if (count <= 1) return;
    if (a.offsets != nullptr)
    {
        bool lower = false;
        for (int64_t i = threadIdx.x; i < n; i += kThreads) lower |= a.offsets[i] > begin;
        if (__syncthreads_or(lower) != 0) return;
    }
    // only the sequence's last segment is shorter; what it leaves matters backward in time alone
    if (threadIdx.x < 2) left[threadIdx.x] = exp(decay_log<A>(a.log_decay, head) * static_cast<double>(threadIdx.x == 0 ? a.segment : end - begin - (count - 1) * a.segment));
    __syncthreads();
    const int64_t state = state_of(a.slots, n, a.state_count, a.bad_index);
    if (state < 0) return;
    const double whole = left[0], tail = left[1];
    const int size = p.dq * p.dv;
    const int64_t step = static_cast<int64_t>(a.heads) * size;
    const int stride = gridDim.y * kThreads;
    for (int i0 = blockIdx.y * kThreads + threadIdx.x; i0 < size; i0 += 2 * stride)
    {
        const bool both = i0 + stride < size;
        const int entry[2] = {i0, both ? i0 + stride : i0};
        double run[2] = {0, 0};
        A *states[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
        {
            const int i = entry[e];
            if (p.initial != nullptr)
            {
                const A *from = static_cast<const A *>(p.initial) + (state * a.heads + head) * size;
                run[e] = p.turned ? from[i % p.dv * p.dq + i / p.dv] : from[i];
            }
            states[e] = static_cast<A *>(p.segment_states) + static_cast<int64_t>(head) * size + i;
        }
        for (int64_t k0 = 0; k0 < count; k0 += kJoin)
        {
            A own[2][kJoin];
#pragma unroll
            for (int k = 0; k < kJoin; ++k)
                if (k0 + k + 1 < count)
                {
                    const int64_t at = segment_state(a, n, begin, reverse ? count - 1 - k0 - k : k0 + k) * step;
                    own[0][k] = states[0][at];
                    own[1][k] = states[1][at];
                }
#pragma unroll
            for (int k = 0; k < kJoin; ++k)
            {
                if (k0 + k >= count) break;
                const int64_t at = reverse ? count - 1 - k0 - k : k0 + k;
                const int64_t place = segment_state(a, n, begin, at) * step;
                states[0][place] = static_cast<A>(run[0]);
                if (both) states[1][place] = static_cast<A>(run[1]);
                if (k0 + k + 1 < count)
                {
                    const double left_over = at == count - 1 ? tail : whole;
                    run[0] = left_over * run[0] + own[0][k];
                    run[1] = left_over * run[1] + own[1][k];
                }
            }
        }
    }
}

struct ShareArgs
{
    const void *sums[2];
    TokenRows out[2];
    int32_t columns[2];
    int32_t heads, group;
    const int64_t *offsets;
    int64_t sequences, tokens;
};

// Rows that a CTA of the share kernel takes at once.
__host__ __device__ __forceinline__ int share_at_once(int heads, int columns) { return heads * columns >= 1024 ? 1 : 1024 / (heads * columns); }

// out[row, h, c] = sum over the query heads of head h, in ascending order: the gradients of shared keys (blockIdx.y = 0) and values, for the
// rows that sequences own.
template <class T>
__global__ void __launch_bounds__(kThreads) attention_share_kernel(const __grid_constant__ ShareArgs a)
{
    using A = typename Element<T>::Acc;
    constexpr int AT_ONCE = 4;
    const A *sums = static_cast<const A *>(blockIdx.y ? a.sums[1] : a.sums[0]);
    const TokenRows &out = blockIdx.y ? a.out[1] : a.out[0];
    const int columns = blockIdx.y ? a.columns[1] : a.columns[0], group = a.group;
    const int each = a.heads * columns, some = share_at_once(a.heads, columns);
    int64_t begin = 0, end = a.sequences * a.tokens, ranges = 1, highest = INT64_MIN;
    bool whole = true;
    if (a.offsets != nullptr)
    {
        // one range from the first sequence to the last, unless some are skipped
        begin = a.offsets[0];
        end = a.offsets[a.sequences];
        whole = offsets_ascend(a.offsets, a.sequences, a.tokens);
        if (!whole) ranges = a.sequences;
    }
    for (int64_t range = 0; range < ranges; ++range)
    {
        if (!whole)
        {
            const bool there = rows_of_sequence(a.offsets, range, a.tokens, highest, begin, end);
            highest = max(highest, begin);
            if (!there) continue;
        }
        for (int64_t first = begin + static_cast<int64_t>(blockIdx.x) * some; first < end; first += static_cast<int64_t>(gridDim.x) * some)
        {
            const int count = static_cast<int>(min(static_cast<int64_t>(some), end - first)) * each;
            for (int i0 = threadIdx.x; i0 < count; i0 += AT_ONCE * kThreads)
            {
                A s[AT_ONCE];
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u) s[u] = 0;
                for (int k = 0; k < group; ++k)
                {
#pragma unroll
                    for (int u = 0; u < AT_ONCE; ++u)
                    {
                        const int i = i0 + u * kThreads, h = i / columns;       // over the heads of all these rows
                        if (i < count) s[u] += sums[((first * a.heads + h) * group + k) * columns + (i - h * columns)];
                    }
                }
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u)
                {
                    const int i = i0 + u * kThreads;
                    if (i >= count) break;
                    const int own = i / each, rest = i - own * each, h = rest / columns, c = rest - h * columns;
                    const int64_t row = first + own, n = a.offsets == nullptr ? row / a.tokens : 0, t = row - n * a.tokens;
                    static_cast<T *>(out.data)[n * out.sequence + t * out.token + h * out.head + c] = narrow<T>(s[u]);
                }
            }
        }
    }
}

struct StepArgs
{
    TokenRows q, k, v, out;             // token: the distance of two requests
    int32_t heads, dk, dv, lanes;       // lanes: threads of one row of the state, a power of two
    int32_t tiles;
    const void *log_decay, *state_in;
    void *state_out;
    const int32_t *slots;
    int64_t requests, state_count;
    double scale;
    int *bad_index;
};

// One token of every request: state <- lam state + k v^T, out = scale q^T state.  Bound by HBM: the state is read and written
// once (8 bytes per entry in 32 bits) for five operations.  A CTA takes one head's state (or a tile of its columns), neighbouring
// lanes neighbouring packs of a row; a thread has UNROLL rows' packs in flight.  The rows' parts of `out` are added per thread,
// then over the lanes of a warp, then over the warps in ascending order.
template <class T, int VN>
__global__ void __launch_bounds__(kThreads) attention_step_kernel(StepArgs a)
{
    using A = typename Element<T>::Acc;
    constexpr int UNROLL = 8;
    __shared__ A sk[kMaxHead], sq[kMaxHead], part[kThreads / 32][32 * VN];
    const int head = blockIdx.x % a.heads, tile = blockIdx.x / a.heads % a.tiles;
    const int64_t n = blockIdx.x / (static_cast<int64_t>(a.heads) * a.tiles);
    const int64_t state = state_of(a.slots, n, a.state_count, a.bad_index);
    if (state < 0) return;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int row0 = threadIdx.x / a.lanes, rows = kThreads / a.lanes;
    const int c = tile * 32 * VN + threadIdx.x % a.lanes * VN;
    const bool there = c < a.dv;
    const int64_t base = (state * a.heads + head) * static_cast<int64_t>(a.dk) * a.dv + c;
    const A *in = static_cast<const A *>(a.state_in) + base;
    A *to = static_cast<A *>(a.state_out) + base;
    Pack<A, VN> s[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i)
    {
        const int d = row0 + i * rows;
        if (there && d < a.dk) s[i] = *reinterpret_cast<const Pack<A, VN> *>(in + static_cast<int64_t>(d) * a.dv);
    }
    const T *q = static_cast<const T *>(a.q.data) + n * a.q.token + static_cast<int64_t>(head / a.q.group) * a.q.head,
            *k = static_cast<const T *>(a.k.data) + n * a.k.token + static_cast<int64_t>(head / a.k.group) * a.k.head,
            *v = static_cast<const T *>(a.v.data) + n * a.v.token + static_cast<int64_t>(head / a.v.group) * a.v.head;
    for (int d = threadIdx.x; d < a.dk; d += kThreads)
    {
        sk[d] = widen(k[d]);
        sq[d] = widen(q[d]);
    }
    const A lam = static_cast<A>(exp(static_cast<double>(decay_log<A>(a.log_decay, head))));
    A x[VN], o[VN];
#pragma unroll
    for (int j = 0; j < VN; ++j)
    {
        x[j] = there ? static_cast<A>(widen(v[c + j])) : A(0);
        o[j] = 0;
    }
    __syncthreads();
    for (int d0 = row0; d0 < a.dk; d0 += UNROLL * rows)
    {
        if (d0 != row0)
        {
#pragma unroll
            for (int i = 0; i < UNROLL; ++i)
            {
                const int d = d0 + i * rows;
                if (there && d < a.dk) s[i] = *reinterpret_cast<const Pack<A, VN> *>(in + static_cast<int64_t>(d) * a.dv);
            }
        }
#pragma unroll
        for (int i = 0; i < UNROLL; ++i)
        {
            const int d = d0 + i * rows;
            if (!there || d >= a.dk) continue;
            const A kd = sk[d], qd = sq[d];
#pragma unroll
            for (int j = 0; j < VN; ++j)
            {
                s[i].x[j] = lam * s[i].x[j] + kd * x[j];
                o[j] += qd * s[i].x[j];
            }
            *reinterpret_cast<Pack<A, VN> *>(to + static_cast<int64_t>(d) * a.dv) = s[i];
        }
    }
#pragma unroll
    for (int j = 0; j < VN; ++j)
        for (int w = a.lanes; w < 32; w <<= 1) o[j] += __shfl_xor_sync(0xffffffffu, o[j], w);
    if (lane < a.lanes)
    {
#pragma unroll
        for (int j = 0; j < VN; ++j) part[warp][lane * VN + j] = o[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.lanes * VN; i += kThreads)
    {
        const int column = tile * 32 * VN + i;
        if (column >= a.dv) continue;
        A sum = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) sum += part[w][i];
        (static_cast<T *>(a.out.data) + n * a.out.token + static_cast<int64_t>(head / a.out.group) * a.out.head)[column] =
            narrow<T>(static_cast<A>(a.scale) * sum);
    }
}

// ---------------------------------------------------------------- host side

constexpr int kSegmentQuantum = 128;    // every kernel's chunk divides it
constexpr int kPlaneTokens = 128;       // fewer tokens stay on the ordinary cores
constexpr int64_t kMaxRows = int64_t(1) << 40;      // of all heads, more than any memory holds: sizes of scratch stay within 64 bits

std::string head_fault(const acro_b200_linear_attention_desc *d, bool packed)
{
    if (d == nullptr) return "null descriptor";
    if (!known_type(d->type)) return "unknown element type";
    if (d->q_heads < 1 || d->kv_heads < 1 || d->q_heads % d->kv_heads != 0) return "q_heads is not a positive multiple of kv_heads";
    if (d->q_heads > 65535) return "more than 65535 heads";
    if (d->dk < 1 || d->dk > kMaxHead || d->dv < 1 || d->dv > kMaxHead) return "head sizes are not in 1 .. 256";
    if (d->sequences < 0 || d->tokens < 0) return "negative number of sequences or tokens";
    const int64_t most = kMaxRows / d->q_heads;
    if (d->tokens > most || d->sequences > most || (!packed && d->sequences > 0 && d->tokens > most / d->sequences)) return "more than 2^40 rows of all heads";
    if (!(d->scale - d->scale == 0)) return "the scale is not finite";
    return "";
}

// Tokens of a segment.  A cut of the sequences into `wanted` segments each makes the GPU's waves of CTAs shorter, and costs a second
// walk over k and v (0.4 of the main pass on the tensor cores, 0.6 on the other path) and the join (as long as 6 chunks of 64 tokens): the cheapest number
// is taken, for the CTAs that an SM holds (tensor-core pass: 1; the other: 2 at least).  Packed sequences are treated as one axis of all
// their rows, since their lengths are not known here; segments of three quarters of that length cost the same over 15 packed shapes, half
// the length 14 % more.  On the tensor cores a segment has 256 tokens at least: 13 shapes took 108 us on average with 512, 93 with 256 (4 x 1024
// tokens of 12 heads in fp32 101 and 88 us), 91 with 128, but a gradient of packed sequences 12 % more than with 256.
int64_t segment_tokens(const acro_b200_linear_attention_desc &d, bool packed, bool tensor_cores, int passes)
{
    const int64_t slots = (sm_count() > 0 ? sm_count() : 148) * (tensor_cores ? 1 : 2);
    const int64_t whole = std::max<int64_t>(1, (d.tokens + kSegmentQuantum - 1) / kSegmentQuantum) * kSegmentQuantum;
    const int64_t pairs = (packed ? 1 : std::max<int64_t>(1, d.sequences)) * d.q_heads * passes;
    const int64_t shortest = kSegmentQuantum * (tensor_cores ? 2 : 1);
    int64_t best = whole;
    double cost = static_cast<double>((pairs + slots - 1) / slots) * whole;
    for (int64_t wanted = 2; wanted <= slots / pairs + 1 && whole / wanted >= shortest; ++wanted)
    {
        const int64_t segment = ((d.tokens + wanted - 1) / wanted + kSegmentQuantum - 1) / kSegmentQuantum * kSegmentQuantum;
        const int64_t each = (d.tokens + segment - 1) / segment;
        const double c = (tensor_cores ? 1.4 : 1.6) * static_cast<double>((pairs * each + slots - 1) / slots) * segment + 6 * 64;
        if (c < cost)
        {
            cost = c;
            best = segment;
        }
    }
    return best;
}

int64_t item_bound(const acro_b200_linear_attention_desc &d, bool packed, int64_t segment)
{
    const int64_t each = d.tokens <= segment ? 1 : (d.tokens + segment - 1) / segment;
    if (!packed) return d.sequences * each;
    return d.tokens <= segment ? d.sequences : d.sequences + d.tokens / segment;
}

bool may_cut(const acro_b200_linear_attention_desc &d, int64_t segment) { return d.tokens > segment; }

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// For whichever path the arrays will turn out to allow.
size_t states_bytes(const acro_b200_linear_attention_desc &d, bool packed, int passes)
{
    size_t most = 0;
    for (int tensor_cores = 0; tensor_cores < 2; ++tensor_cores)
    {
        const int64_t segment = segment_tokens(d, packed, tensor_cores != 0, passes);
        if (may_cut(d, segment) && (tensor_cores == 0 || d.type != ACRO_B200_F64))
            most = std::max(most, round256(static_cast<size_t>(states_of_segments(d.sequences, d.tokens, segment, packed)) * d.q_heads * d.dk * d.dv * statistic_bytes(d.type)));
    }
    return most;
}

size_t shared_bytes(const acro_b200_linear_attention_desc &d, bool packed, int columns)
{
    if (d.q_heads == d.kv_heads) return 0;
    const int64_t rows = packed ? d.tokens : d.sequences * d.tokens;
    return round256(static_cast<size_t>(rows) * d.q_heads * columns * statistic_bytes(d.type));
}

// Do two arrays of states share memory without being the same?  A sequence's state would be written while another one's is still read.
bool states_cross(const acro_b200_linear_attention_desc &d, int64_t count, const void *x, const void *y)
{
    if (x == nullptr || y == nullptr || x == y) return false;
    const __int128 bytes = static_cast<__int128>(count) * d.q_heads * d.dk * d.dv * static_cast<int64_t>(statistic_bytes(d.type));
    const __int128 apart = static_cast<__int128>(reinterpret_cast<uintptr_t>(x)) - reinterpret_cast<uintptr_t>(y);
    return apart < bytes && -apart < bytes;
}

TokenRows rows_from(const acro_b200_token_array &x, int group) { return {x.data, x.sequence_stride, x.token_stride, x.head_stride, group}; }

// Does no row of an array share an entry with another?  Of heads, tokens and sequences the one of a larger stride has to stride over all of
// the smaller ones.
bool rows_apart(const acro_b200_token_array &x, int64_t columns, int heads, int64_t tokens, int64_t sequences, bool packed)
{
    struct { int64_t stride, count; } dims[3] = {{x.head_stride, heads}, {x.token_stride, tokens}, {x.sequence_stride, packed ? 1 : sequences}};
    std::sort(dims, dims + 3, [](const auto &a, const auto &b) { return a.stride < b.stride; });
    __int128 extent = columns;
    for (const auto &dim : dims)
    {
        if (dim.count <= 1) continue;
        if (dim.stride < extent) return false;
        extent += static_cast<__int128>(dim.stride) * (dim.count - 1);
    }
    return true;
}

// `written`: by different CTAs, so no two rows may share an entry; rows that are only read are as far apart as their columns in each dimension.
std::string array_fault(const acro_b200_linear_attention_desc &d, const acro_b200_token_array *x, int64_t columns, int heads, int64_t tokens, int64_t sequences,
                        bool packed, const char *name, bool written = false)
{
    const std::string n(name);
    if (x == nullptr || x->data == nullptr) return n + " is a null pointer";
    if ((heads > 1 && x->head_stride < columns) || (tokens > 1 && x->token_stride < columns) || (!packed && sequences > 1 && x->sequence_stride < columns) ||
        (written && !rows_apart(*x, columns, heads, tokens, sequences, packed)))
        return n + " has rows that overlap";
    if (!aligned_to({x->data}, element_bytes(d.type))) return n + " is not aligned to its elements";
    return "";
}

// Do the pass's operands come in packs of 16 bytes of sums?
template <class T>
bool rows_in_packs(const AttentionPass &p)
{
    constexpr int n = 16 / sizeof(typename Element<T>::Acc);
    const auto fits = [](const TokenRows &r, int columns) {
        return reinterpret_cast<uintptr_t>(r.data) % (n * sizeof(T)) == 0 && r.sequence % n == 0 && r.token % n == 0 && r.head % n == 0 && columns % n == 0;
    };
    return fits(p.q, p.dq) && fits(p.k, p.dq) && fits(p.v, p.dv);
}

template <class T, int C, int SV>
int run_pass_tiled(const AttentionArgs &all, bool states_only, cudaStream_t stream)
{
    AttentionArgs a = all;
    int slices = 1;
    size_t smem = 0;
    for (int i = 0; i < a.passes; ++i)
    {
        a.pass[i].packs = rows_in_packs<T>(a.pass[i]);
        slices = std::max(slices, (a.pass[i].dv + SV - 1) / SV);
        smem = std::max(smem, pass_smem_bytes<typename Element<T>::Acc, C, SV>(a.pass[i].dq));
    }
    cudaError_t status = allow_dynamic_smem(attention_pass_kernel<T, C, SV>, smem);
    if (status != cudaSuccess) return fail_cuda(status, "acro_b200_linear_attention");
    const int64_t grid = a.items * a.heads * slices;
    if (grid > INT32_MAX) return fail_unsupported("acro_b200_linear_attention: more than 2^31 segments x heads");
    attention_pass_kernel<T, C, SV><<<dim3(static_cast<unsigned>(grid), a.passes), kThreads, smem, stream>>>(a, slices, states_only);
    return launch_status("acro_b200_linear_attention");
}

// The scores are made anew for every slice of v's columns, so heads of more than 64 columns take slices of 128, with half the tokens a
// chunk to make room.
template <class T>
int run_pass(const AttentionArgs &a, bool states_only, cudaStream_t stream)
{
    if constexpr (sizeof(T) == 8) return run_pass_tiled<T, 32, 32>(a, states_only, stream);
    else
    {
        int widest = 0;
        for (int i = 0; i < a.passes; ++i) widest = std::max(widest, a.pass[i].dv);
        return widest <= 64 ? run_pass_tiled<T, 64, 64>(a, states_only, stream) : run_pass_tiled<T, 32, 128>(a, states_only, stream);
    }
}

int run_pass_of(int type, const AttentionArgs &a, bool tensor_cores, bool states_only, cudaStream_t stream)
{
    if (tensor_cores) return attention_mma_launch(a, type, states_only, stream);
    switch (type)
    {
    case ACRO_B200_F64: return run_pass<double>(a, states_only, stream);
    case ACRO_B200_F32: return run_pass<float>(a, states_only, stream);
    case ACRO_B200_BF16: return run_pass<__nv_bfloat16>(a, states_only, stream);
    default: return run_pass<__half>(a, states_only, stream);
    }
}

// Do inputs of these sizes go to the tensor cores as planes of bf16 parts?  fp64 has none; bf16 rows of a multiple of eight columns are
// read as they are (and stay on the other path if they are not aligned).  A few tokens are not worth the planes.
bool takes_planes(const acro_b200_linear_attention_desc &d)
{
    if (d.type == ACRO_B200_F64 || d.dk > 128 || d.dv > 128 || d.tokens < kPlaneTokens) return false;
    return d.type != ACRO_B200_BF16 || d.dk % 8 != 0 || d.dv % 8 != 0;
}

size_t planes_bytes(const acro_b200_linear_attention_desc &d, bool packed, bool gradient)
{
    if (!takes_planes(d)) return 0;
    const int64_t rows = packed ? d.tokens : d.sequences * d.tokens;
    return attention_planes_bytes(d.type, rows, d.q_heads, d.dk) + attention_planes_bytes(d.type, rows, d.kv_heads, d.dk) +
           attention_planes_bytes(d.type, rows, d.kv_heads, d.dv) + (gradient ? attention_planes_bytes(d.type, rows, d.q_heads, d.dv) : 0);
}

// `arrays`: q, k, v (and dout) as the passes use them; `planes`: scratch of planes_bytes.
int run_all(const acro_b200_linear_attention_desc &d, AttentionArgs &a, const TokenRows *arrays, const int *columns, int count, void *planes,
            cudaStream_t stream)
{
    const bool packed = a.offsets != nullptr, sizes = d.type != ACRO_B200_F64 && attention_mma_sizes(a);
    const bool direct = sizes && d.type == ACRO_B200_BF16 && attention_mma_direct(a), tensor_cores = direct || (sizes && takes_planes(d));
    if (tensor_cores && !direct)
    {
        const int status = attention_split(a, d.type, arrays, columns, count, planes, stream);
        if (status != ACRO_B200_OK) return status;
    }
    a.segment = segment_tokens(d, packed, tensor_cores, a.passes);
    a.items = item_bound(d, packed, a.segment);
    if (may_cut(d, a.segment))
    {
        int status = run_pass_of(d.type, a, tensor_cores, true, stream);
        if (status != ACRO_B200_OK) return status;
        int64_t entries = 0;
        for (int i = 0; i < a.passes; ++i) entries = std::max<int64_t>(entries, static_cast<int64_t>(a.pass[i].dq) * a.pass[i].dv);
        const dim3 grid(static_cast<unsigned>(a.sequences * a.heads), static_cast<unsigned>(std::min<int64_t>(32, (entries + 2 * kThreads - 1) / (2 * kThreads))),
                        a.passes);
        if (d.type == ACRO_B200_F64) attention_join_kernel<double><<<grid, kThreads, 0, stream>>>(a);
        else attention_join_kernel<float><<<grid, kThreads, 0, stream>>>(a);
        status = launch_status("acro_b200_linear_attention");
        if (status != ACRO_B200_OK) return status;
    }
    return run_pass_of(d.type, a, tensor_cores, false, stream);
}

int common_args(const acro_b200_linear_attention_desc &d, const void *log_decay, const int64_t *offsets, AttentionArgs *a)
{
    a->heads = d.q_heads;
    a->log_decay = log_decay;
    a->offsets = offsets;
    a->slots = nullptr;
    a->state_count = d.sequences;
    a->sequences = d.sequences;
    a->tokens = d.tokens;
    a->bad_index = bad_index_flag_device_ptr();
    a->wait_flag = wait_flag_device_ptr();
    if (a->bad_index == nullptr || a->wait_flag == nullptr) return fail_cuda(cudaErrorUnknown, "acro_b200_linear_attention (device flag)");
    if (d.sequences * d.q_heads > INT32_MAX) return fail_unsupported("acro_b200_linear_attention: more than 2^31 sequences x heads");
    return ACRO_B200_OK;
}

}

extern "C" {

size_t acro_b200_linear_attention_scratch_bytes(const acro_b200_linear_attention_desc *desc, int packed)
{
    if (!head_fault(desc, packed != 0).empty()) return 0;
    return states_bytes(*desc, packed != 0, 1) + planes_bytes(*desc, packed != 0, false);
}

int acro_b200_linear_attention(const acro_b200_linear_attention_desc *desc, const acro_b200_token_array *q, const acro_b200_token_array *k,
                               const acro_b200_token_array *v, const acro_b200_token_array *out, const void *log_decay, const int64_t *offsets,
                               const void *initial_state, void *final_state, const int32_t *slots, int64_t state_count, void *scratch, size_t scratch_bytes,
                               void *stream)
{
    const std::string name = "acro_b200_linear_attention: ";
    std::string fault = head_fault(desc, offsets != nullptr);
    if (!fault.empty()) return fail_invalid(name + fault);
    const acro_b200_linear_attention_desc &d = *desc;
    if (d.sequences == 0) return ACRO_B200_OK;
    const bool packed = offsets != nullptr, rows = d.tokens > 0;
    if (rows)
    {
        if (fault.empty()) fault = array_fault(d, q, d.dk, d.q_heads, d.tokens, d.sequences, packed, "q");
        if (fault.empty()) fault = array_fault(d, k, d.dk, d.kv_heads, d.tokens, d.sequences, packed, "k");
        if (fault.empty()) fault = array_fault(d, v, d.dv, d.kv_heads, d.tokens, d.sequences, packed, "v");
        if (fault.empty()) fault = array_fault(d, out, d.dv, d.q_heads, d.tokens, d.sequences, packed, "out", true);
    }
    if (fault.empty() && log_decay == nullptr) fault = "log_decay is a null pointer";
    if (fault.empty() && slots != nullptr && state_count < 0) fault = "negative state_count";
    if (fault.empty() && slots == nullptr && state_count != d.sequences && (initial_state != nullptr || final_state != nullptr))
        fault = "without slots there is one state per sequence";
    const size_t states = states_bytes(d, packed, 1), need = states + planes_bytes(d, packed, false);
    if (fault.empty() && need > 0 && (scratch == nullptr || scratch_bytes < need || !aligned16(scratch)))
        fault = "scratch is smaller than acro_b200_linear_attention_scratch_bytes or not 16-byte aligned";
    if (fault.empty() && (!aligned_to({log_decay, initial_state, final_state}, statistic_bytes(d.type)) || !aligned_to({offsets}, 8) || !aligned_to({slots}, 4)))
        fault = "log_decay, offsets, slots or a state is not aligned to its elements";
    if (fault.empty() && rows && (out->data == q->data || out->data == k->data || out->data == v->data))
        fault = "out takes the place of an operand that is still read";
    if (fault.empty() && states_cross(d, state_count, initial_state, final_state)) fault = "final_state overlaps initial_state without being the same";
    if (fault.empty() && ((rows && !all_on_device({q->data, k->data, v->data, out->data})) ||
                          !all_on_device({log_decay, offsets, slots, initial_state, final_state, need > 0 ? scratch : nullptr})))
        fault = "an array, log_decay, offsets, slots, a state or scratch is not memory of the current device";
    if (!fault.empty()) return fail_invalid(name + fault);
    AttentionArgs a = {};
    int status = common_args(d, log_decay, offsets, &a);
    if (status != ACRO_B200_OK) return status;
    if (slots != nullptr)
    {
        a.slots = slots;
        // without states the slots only say which sequences are there
        a.state_count = initial_state != nullptr || final_state != nullptr ? state_count : int64_t(INT32_MAX) + 1;
    }
    const acro_b200_token_array none = {};
    const int group = d.q_heads / d.kv_heads;
    a.passes = 1;
    AttentionPass &p = a.pass[0];
    p.q = rows_from(rows ? *q : none, 1);
    p.k = rows_from(rows ? *k : none, group);
    p.v = rows_from(rows ? *v : none, group);
    p.out = rows_from(rows ? *out : none, 1);
    p.dq = d.dk;
    p.dv = d.dv;
    p.state_scale = 1;
    p.out_scale = d.scale;
    p.initial = initial_state;
    p.final = final_state;
    p.segment_states = scratch;
    const TokenRows arrays[3] = {p.q, p.k, p.v};
    const int columns[3] = {d.dk, d.dk, d.dv};
    return run_all(d, a, arrays, columns, 3, static_cast<unsigned char *>(scratch) + states, as_stream(stream));
}

int acro_b200_linear_attention_step(const acro_b200_linear_attention_desc *desc, const acro_b200_token_array *q, const acro_b200_token_array *k,
                                    const acro_b200_token_array *v, const acro_b200_token_array *out, const void *log_decay, const void *state_in,
                                    void *state_out, const int32_t *slots, int64_t state_count, void *stream)
{
    const std::string name = "acro_b200_linear_attention_step: ";
    std::string fault = head_fault(desc, false);
    if (!fault.empty()) return fail_invalid(name + fault);
    const acro_b200_linear_attention_desc &d = *desc;
    if (d.tokens != 1) return fail_invalid(name + "a step takes one token of each sequence");
    if (d.sequences == 0) return ACRO_B200_OK;
    // the distance of two requests is that of two sequences
    fault = array_fault(d, q, d.dk, d.q_heads, 1, d.sequences, false, "q");
    if (fault.empty()) fault = array_fault(d, k, d.dk, d.kv_heads, 1, d.sequences, false, "k");
    if (fault.empty()) fault = array_fault(d, v, d.dv, d.kv_heads, 1, d.sequences, false, "v");
    if (fault.empty()) fault = array_fault(d, out, d.dv, d.q_heads, 1, d.sequences, false, "out", true);
    if (fault.empty() && (log_decay == nullptr || state_in == nullptr || state_out == nullptr)) fault = "null pointer";
    if (fault.empty() && (!aligned_to({log_decay, state_in, state_out}, statistic_bytes(d.type)) || !aligned_to({slots}, 4)))
        fault = "log_decay, slots or a state is not aligned to its elements";
    if (fault.empty() && (out->data == q->data || out->data == k->data || out->data == v->data))
        fault = "out takes the place of an operand that is still read";
    if (fault.empty() && (state_count < 0 || (slots == nullptr && state_count != d.sequences))) fault = "without slots there is one state per sequence";
    if (fault.empty() && states_cross(d, state_count, state_in, state_out)) fault = "state_out overlaps state_in without being the same";
    if (fault.empty() && !all_on_device({q->data, k->data, v->data, out->data, log_decay, state_in, state_out, slots}))
        fault = "an array, log_decay, slots or a state is not memory of the current device";
    if (!fault.empty()) return fail_invalid(name + fault);
    StepArgs a = {};
    const int group = d.q_heads / d.kv_heads;
    a.q = rows_from(*q, 1);
    a.k = rows_from(*k, group);
    a.v = rows_from(*v, group);
    a.out = rows_from(*out, 1);
    a.q.token = q->sequence_stride;
    a.k.token = k->sequence_stride;
    a.v.token = v->sequence_stride;
    a.out.token = out->sequence_stride;
    a.heads = d.q_heads;
    a.dk = d.dk;
    a.dv = d.dv;
    a.log_decay = log_decay;
    a.state_in = state_in;
    a.state_out = state_out;
    a.slots = slots;
    a.requests = d.sequences;
    a.state_count = state_count;
    a.scale = d.scale;
    a.bad_index = bad_index_flag_device_ptr();
    if (a.bad_index == nullptr) return fail_cuda(cudaErrorUnknown, "acro_b200_linear_attention_step (device flag)");
    // packs of 16 bytes when every row of the states starts on their boundary
    const int pack = static_cast<int>(16 / statistic_bytes(d.type));
    const bool packs = d.dv % pack == 0 && aligned16(state_in) && aligned16(state_out);
    const int columns = 32 * (packs ? pack : 1), per_row = (std::min(d.dv, columns) + (packs ? pack : 1) - 1) / (packs ? pack : 1);
    a.tiles = (d.dv + columns - 1) / columns;
    a.lanes = 1;
    while (a.lanes < per_row) a.lanes *= 2;
    const int64_t grid = d.sequences * d.q_heads * a.tiles;
    if (grid > INT32_MAX) return fail_unsupported(name + "more than 2^31 requests x heads");
    const unsigned g = static_cast<unsigned>(grid);
    cudaStream_t st = as_stream(stream);
    switch (d.type)
    {
    case ACRO_B200_F64:
        if (packs) attention_step_kernel<double, 2><<<g, kThreads, 0, st>>>(a);
        else attention_step_kernel<double, 1><<<g, kThreads, 0, st>>>(a);
        break;
    case ACRO_B200_F32:
        if (packs) attention_step_kernel<float, 4><<<g, kThreads, 0, st>>>(a);
        else attention_step_kernel<float, 1><<<g, kThreads, 0, st>>>(a);
        break;
    case ACRO_B200_BF16:
        if (packs) attention_step_kernel<__nv_bfloat16, 4><<<g, kThreads, 0, st>>>(a);
        else attention_step_kernel<__nv_bfloat16, 1><<<g, kThreads, 0, st>>>(a);
        break;
    default:
        if (packs) attention_step_kernel<__half, 4><<<g, kThreads, 0, st>>>(a);
        else attention_step_kernel<__half, 1><<<g, kThreads, 0, st>>>(a);
    }
    return launch_status("acro_b200_linear_attention_step");
}

size_t acro_b200_linear_attention_backward_scratch_bytes(const acro_b200_linear_attention_desc *desc, int packed)
{
    if (!head_fault(desc, packed != 0).empty()) return 0;
    return 3 * states_bytes(*desc, packed != 0, 3) + shared_bytes(*desc, packed != 0, desc->dk) + shared_bytes(*desc, packed != 0, desc->dv) +
           planes_bytes(*desc, packed != 0, true);
}

int acro_b200_linear_attention_backward(const acro_b200_linear_attention_desc *desc, const acro_b200_token_array *q, const acro_b200_token_array *k,
                                        const acro_b200_token_array *v, const acro_b200_token_array *dout, const void *log_decay, const int64_t *offsets,
                                        const void *initial_state, const void *d_final_state, const acro_b200_token_array *dq,
                                        const acro_b200_token_array *dk, const acro_b200_token_array *dv, void *d_initial_state, void *scratch,
                                        size_t scratch_bytes, void *stream)
{
    const std::string name = "acro_b200_linear_attention_backward: ";
    std::string fault = head_fault(desc, offsets != nullptr);
    if (!fault.empty()) return fail_invalid(name + fault);
    const acro_b200_linear_attention_desc &d = *desc;
    if (d.sequences == 0) return ACRO_B200_OK;
    const bool packed = offsets != nullptr, rows = d.tokens > 0;
    const struct { const acro_b200_token_array *x; int columns, heads; const char *name; bool written; } given[] = {
        {q, d.dk, d.q_heads, "q", false}, {k, d.dk, d.kv_heads, "k", false}, {v, d.dv, d.kv_heads, "v", false}, {dout, d.dv, d.q_heads, "dout", false},
        {dq, d.dk, d.q_heads, "dq", true}, {dk, d.dk, d.kv_heads, "dk", true}, {dv, d.dv, d.kv_heads, "dv", true}};
    if (rows)
        for (const auto &x : given)
            if (fault.empty()) fault = array_fault(d, x.x, x.columns, x.heads, d.tokens, d.sequences, packed, x.name, x.written);
    if (fault.empty() && log_decay == nullptr) fault = "log_decay is a null pointer";
    const size_t need = acro_b200_linear_attention_backward_scratch_bytes(desc, packed);
    if (fault.empty() && need > 0 && (scratch == nullptr || scratch_bytes < need || !aligned16(scratch)))
        fault = "scratch is smaller than acro_b200_linear_attention_backward_scratch_bytes or not 16-byte aligned";
    if (fault.empty() && (!aligned_to({log_decay, initial_state, d_final_state, d_initial_state}, statistic_bytes(d.type)) || !aligned_to({offsets}, 8)))
        fault = "log_decay, offsets or a state is not aligned to its elements";
    if (fault.empty() && d_initial_state != nullptr &&
        (d_initial_state == d_final_state || d_initial_state == initial_state || states_cross(d, d.sequences, d_initial_state, d_final_state) ||
         states_cross(d, d.sequences, d_initial_state, initial_state)))
        fault = "d_initial_state takes the place of a state that is still read";
    if (fault.empty() && rows)
        for (const acro_b200_token_array *to : {dq, dk, dv})
            for (const acro_b200_token_array *from : {q, k, v, dout})
                if (to->data == from->data) fault = "a gradient takes the place of an operand that is still read";
    if (fault.empty() && rows && (dq->data == dk->data || dq->data == dv->data || dk->data == dv->data)) fault = "two gradients take the same place";
    if (fault.empty() && rows)
        for (const auto &x : given)
            if (!all_on_device({x.x->data})) fault = std::string(x.name) + " is not memory of the current device";
    if (fault.empty() && !all_on_device({log_decay, offsets, initial_state, d_final_state, d_initial_state, need > 0 ? scratch : nullptr}))
        fault = "log_decay, offsets, a state or scratch is not memory of the current device";
    if (!fault.empty()) return fail_invalid(name + fault);
    AttentionArgs a = {};
    int status = common_args(d, log_decay, offsets, &a);
    if (status != ACRO_B200_OK) return status;
    const acro_b200_token_array none = {};
    const int group = d.q_heads / d.kv_heads;
    const TokenRows rq = rows_from(rows ? *q : none, 1), rk = rows_from(rows ? *k : none, group), rv = rows_from(rows ? *v : none, group),
                    ro = rows_from(rows ? *dout : none, 1);
    const size_t states = states_bytes(d, packed, 3);
    unsigned char *at = static_cast<unsigned char *>(scratch);
    a.passes = 3;
    for (int i = 0; i < 3; ++i)
    {
        AttentionPass &p = a.pass[i];
        p.segment_states = at;
        at += states;
        p.reverse = i > 0;
        p.state_scale = i > 0 ? d.scale : 1;
        p.out_scale = i > 0 ? 1 : d.scale;
        p.turned = i < 2;
        p.dq = i < 2 ? d.dv : d.dk;
        p.dv = i < 2 ? d.dk : d.dv;
        p.initial = i > 0 ? d_final_state : initial_state;
        p.final = i == 2 ? d_initial_state : nullptr;
    }
    a.pass[0].q = ro;
    a.pass[0].k = rv;
    a.pass[0].v = rk;
    a.pass[0].out = rows_from(rows ? *dq : none, 1);
    a.pass[1].q = rv;
    a.pass[1].k = ro;
    a.pass[1].v = rq;
    a.pass[2].q = rk;
    a.pass[2].k = rq;
    a.pass[2].v = ro;
    const TokenRows arrays[4] = {rq, rk, rv, ro};
    const int columns[4] = {d.dk, d.dk, d.dv, d.dv};
    if (group == 1)
    {
        a.pass[1].out = rows_from(rows ? *dk : none, 1);
        a.pass[2].out = rows_from(rows ? *dv : none, 1);
        return run_all(d, a, arrays, columns, 4, at, as_stream(stream));
    }
    // a row of sums per query head, added up afterwards
    ShareArgs both = {{nullptr, nullptr}, {rows_from(rows ? *dk : none, 1), rows_from(rows ? *dv : none, 1)}, {d.dk, d.dv}, d.kv_heads, group, offsets, d.sequences,
                      d.tokens};
    for (int i = 0; i < 2; ++i)
    {
        both.sums[i] = at;
        const int64_t row = static_cast<int64_t>(d.q_heads) * both.columns[i];
        a.pass[1 + i].out = {at, row * d.tokens, row, both.columns[i], 1};
        a.pass[1 + i].sums = 1;
        at += shared_bytes(d, packed, both.columns[i]);
    }
    cudaStream_t st = as_stream(stream);
    status = run_all(d, a, arrays, columns, 4, at, st);
    if (status != ACRO_B200_OK || !rows) return status;
    const int some = std::min(share_at_once(d.kv_heads, d.dk), share_at_once(d.kv_heads, d.dv));
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(((packed ? 1 : d.sequences) * d.tokens + some - 1) / some, 148 * 8)), 2);
    switch (d.type)
    {
    case ACRO_B200_F64: attention_share_kernel<double><<<grid, kThreads, 0, st>>>(both); break;
    case ACRO_B200_F32: attention_share_kernel<float><<<grid, kThreads, 0, st>>>(both); break;
    case ACRO_B200_BF16: attention_share_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(both); break;
    default: attention_share_kernel<__half><<<grid, kThreads, 0, st>>>(both);
    }
    return launch_status("acro_b200_linear_attention_backward");
}

}
