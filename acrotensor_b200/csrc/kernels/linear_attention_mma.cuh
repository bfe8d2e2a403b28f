// Linear attention's pass on the tcgen05 tensor cores, for heads of up to 128 columns.
//
// A CTA walks one segment of one head in chunks of 64 tokens (r, s: tokens of the chunk; a: columns of q and k; b: of v):
//   scores  P[r][s]     = Q[r][a] K[s][a]                            M = r (64 of 128 lanes used)
//   near    O'[b][r]    = V[s][b] P~[r][s]                           P~: scores times powers of the decay and the scales, zero where masked
//   far     O"[b][r]    = S[b][a] Q[r][a]                            S: the state before the chunk, A operand in tensor memory
//   change  D[b][a]     = V[s][b] K~[s][a]                           K~: rows of K times what the decay leaves of them and the state's scale
//   out[r][b] = O' + out_scale come_r O",   S <- lam^m S + D
// The transposed forms put b on the 128 lanes: the state stays in registers (fp32), one row of S^T per thread and a quarter of its
// columns, and becomes an A operand by a store into tensor memory, without a way through shared memory.
//
// Precision: accumulators and the state are fp32; every operand is a sum of bf16 parts (8 bits each).  Inputs: IN parts, 1 for bf16, 2 for
// fp16 (exact) and 3 for fp32 (2^-26).  P~, S and K~: 3 parts whatever the inputs, so that scores and states have on their way into a product
// the bits that they have in fp32 (with two parts of P~ and S, 2^-18, a few bf16 results in ten thousand were rounded the other way; a chunk of
// 128 columns took 2.75 us where it takes 3.07 with three, of 64 columns 1.71 and 2.06).  Of the products of parts those are left out that lie
// below 2^-24 of the whole.  The small ones are multiplied first: the tensor cores' additions lose up to a step of the sum so far, so fewer
// of them happen at its full size; and no sum of theirs spans more
// than a chunk (spanning a segment of 58 cost the final state a digit).
//
// Bound, for bf16 and 128 columns: by HBM 64 KB a chunk, about 2850 cycles of an SM at its share of 6.5 TB/s.  Shared memory comes first:
// the products' operands take about 2370 cycles of it (48 cycles for 64 columns with both operands there, measured alone), copies, K~, P~ and
// stores 2170, of the 5500 cycles (3.07 us) that a chunk takes with all SMs at work.  64 columns: 2.06 us a chunk.  The roles overlap: one
// warp issues copies and products, eight convert operands, sixteen keep the state and write; waiting warps sleep on barriers, one arrival
// a warp; loops are short (the instruction cache held the first versions back).
#ifndef ACRO_B200_KERNELS_LINEAR_ATTENTION_MMA_CUH
#define ACRO_B200_KERNELS_LINEAR_ATTENTION_MMA_CUH

#include "linear_attention.cuh"
#include "umma.cuh"

#include <algorithm>
#include <cuda.h>
#include <type_traits>

using namespace acro_b200_detail;

namespace
{

constexpr int kChunk = 64;
constexpr int kBox = kChunk * 128;          // bytes of 64 rows of 64 columns
// Warps 0 .. 15 keep the state and write `out` (a quarter of the state's columns and of the chunk's rows each, for 32 lanes).
// Warps 16 .. 23 make operands: those on tensor memory lanes 0 .. 63 the weights, the others K~.  Warp 24 issues copies and products.
constexpr int kStateWarps = 16, kOperandWarps = 8, kIssueWarp = kStateWarps + kOperandWarps, kBlock = (kIssueWarp + 1) * 32;
constexpr int kRing = 16;                   // slots of the flags that tell of non-finite values; operand warps run at most 5 chunks ahead

// Columns of tensor memory; the state's parts stand behind the change.
constexpr uint32_t kScores = 0, kNear = 64, kFar = 128, kDelta = 192, kColumns = 512;
constexpr int kSmem = 227 * 1024;           // of a CTA

struct Maps
{
    CUtensorMap q[3], k[3], v[3];
    int32_t sequences;                      // part p of sequence n is number p * sequences + n of a map
};

// NQ, NV: boxes of 64 columns of q and k, of v; IN: parts of an input.
template <int NQ, int NV, int IN>
struct Layout
{
    static constexpr int kParts = 3;                            // of P~ and S
    static constexpr int kQ = 0, kK = IN * NQ * kBox, kV = 2 * IN * NQ * kBox, kStage = IN * (2 * NQ + NV) * kBox;
    static constexpr int kFits = (kSmem - (3 * NQ + kParts) * kBox - 4096) / kStage;
    static constexpr int kStages = kFits < (NQ == 2 ? 3 : 4) ? kFits : NQ == 2 ? 3 : 4;
    static constexpr int kScaled = kStages * kStage;            // K~, three parts
    static constexpr int kWeights = kScaled + 3 * NQ * kBox;    // P~
    static constexpr int kTables = kWeights + kParts * kBox;
    // a first product of M = 128 reads 64 rows behind a box: they lie inside the allocation
    static constexpr int kBytes = kTables + 2048;
    static constexpr int kDynamic = kBytes + 1024;              // the base is rounded up to 1024
    static constexpr uint32_t kState = kDelta + NQ * 64;        // tensor memory
    static_assert(kStages >= 1 && kState + kParts * NQ * 32 <= kColumns, "it fits");
};

struct Shared
{
    float left[kChunk + 4];                 // lam^n times the state's scale: what is left of a token that n tokens follow
    float weight[2 * kChunk];               // of tokens kChunk - i apart, times both scales; zero for those not seen
    alignas(16) float come[2][kChunk];      // what is left at row r of the state before a whole chunk, and before one of length % kChunk
                                            // tokens, times the output's scale
    int odd[kRing];
    uint32_t tmem;
    uint64_t full[4], ready[4], scores, weights, state, out, out_free, change, change_free, drained;
};

// The next bf16 part of x: returns it and leaves the remainder.  Parts of fp32 values above the largest bf16 are finite; an infinity stands
// in the last part (pack_bf16), a NaN in all.
__device__ __forceinline__ uint32_t take_part(Two &x)
{
    const uint32_t part = pack_bf16_finite(x);
    x = sub2(x, unpack_bf16(part));
    return part;
}

__device__ __forceinline__ bool odd_half(uint32_t x) { return (x & 0x7f80u) == 0x7f80u; }
__device__ __forceinline__ bool odd_pair(uint32_t x) { return odd_half(x) || odd_half(x >> 16); }
// The pair with zeros in the place of infinities and NaN.
__device__ __forceinline__ uint32_t finite_pair(uint32_t x) { return (odd_half(x) ? 0u : x & 0xffffu) | (odd_half(x >> 16) ? 0u : x & 0xffff0000u); }

// One arrival for the whole warp, after all its lanes have come here.
__device__ __forceinline__ void warp_arrive(uint64_t *bar)
{
    __syncwarp();
    if (threadIdx.x % 32 == 0) mbar_arrive(bar);
}

__device__ __forceinline__ bool all_wait(uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_asleep(bar, parity)); }

// The products of parts of A and B: the pairs (part i of A, part j of B) with i + j < 3, the small ones first.  `later`: not the first pair.
template <int PA, int PB, class F>
__device__ __forceinline__ void for_pairs(F &&issue)
{
    bool later = false;
#pragma unroll
    for (int sum = 2; sum >= 0; --sum)
#pragma unroll
        for (int i = 0; i <= sum; ++i)
            if (i < PA && sum - i < PB)
            {
                issue(i, sum - i, later);
                later = true;
            }
}

// Two results to rows `to` and `after` of the output's type.
__device__ __forceinline__ void put_two(float *to, float *after, Two o, bool first, bool second)
{
    if (first) *to = first_of(o);
    if (second) *after = second_of(o);
}
__device__ __forceinline__ void put_two(__nv_bfloat16 *to, __nv_bfloat16 *after, Two o, bool first, bool second)
{
    const uint32_t both = narrow2<__nv_bfloat16>(o);
    if (first) *reinterpret_cast<uint16_t *>(to) = static_cast<uint16_t>(both);
    if (second) *reinterpret_cast<uint16_t *>(after) = static_cast<uint16_t>(both >> 16);
}
__device__ __forceinline__ void put_two(__half *to, __half *after, Two o, bool first, bool second)
{
    const uint32_t both = narrow2<__half>(o);
    if (first) *reinterpret_cast<uint16_t *>(to) = static_cast<uint16_t>(both);
    if (second) *reinterpret_cast<uint16_t *>(after) = static_cast<uint16_t>(both >> 16);
}

template <int NQ, int NV, int IN, class OUT>
__global__ void __launch_bounds__(kBlock, 1) attention_mma_kernel(const __grid_constant__ AttentionArgs a, const __grid_constant__ Maps maps)
{
    using L = Layout<NQ, NV, IN>;
    constexpr int PART = NQ * 16;               // columns of the state per thread
    constexpr int SP = L::kParts;
    const int pass = blockIdx.y;
    const AttentionPass &p = a.pass[pass];
    const int head = blockIdx.x % a.heads;
    const int64_t item_index = blockIdx.x / a.heads;
    const bool reverse = p.reverse != 0;
    const SegmentItem item = find_item(a, item_index, reverse);
    if (item.sequence < 0) return;
    const bool cut = segments_of(item.sequence_end - item.sequence_begin, a.segment) > 1;

    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    Shared &sh = *reinterpret_cast<Shared *>(smem + L::kTables);
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x / 32), 0), lane = threadIdx.x % 32;

    const double g = decay_log<float>(a.log_decay, head);
    const int length = static_cast<int>(item.end - item.begin);
    if (threadIdx.x < 2 * kChunk)
    {
        const int i = threadIdx.x, r = i % kChunk, near = reverse ? i - kChunk : kChunk - i, come = reverse ? (i < kChunk ? kChunk : length % kChunk) - 1 - r : r + 1;
        if (i <= kChunk) sh.left[i] = static_cast<float>(exp(g * i) * p.state_scale);
        sh.weight[i] = near >= 0 ? static_cast<float>(exp(g * near) * p.state_scale * p.out_scale) : 0.0f;
        sh.come[i / kChunk][r] = come >= 0 ? static_cast<float>(exp(g * come) * p.out_scale) : 0.0f;
    }
    if (threadIdx.x < kRing) sh.odd[threadIdx.x] = 0;
    if (threadIdx.x == 0)
    {
        for (int i = 0; i < L::kStages; ++i)
        {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.ready[i], kOperandWarps);
        }
        mbar_init(&sh.scores, 1);
        mbar_init(&sh.out, 1);
        mbar_init(&sh.change, 1);
        mbar_init(&sh.drained, 1);
        mbar_init(&sh.weights, kOperandWarps / 2);
        mbar_init(&sh.state, kStateWarps);
        mbar_init(&sh.out_free, kStateWarps);
        mbar_init(&sh.change_free, kStateWarps);
        fence_mbar_init();
    }
    if (warp == kIssueWarp) tmem_alloc(&sh.tmem, kColumns);
    tmem_fence_before_sync();
    __syncthreads();
    tmem_fence_after_sync();
    // All columns are allocated, so the allocation starts at column zero and addresses are constants.
    constexpr uint32_t tmem = 0;
    const int chunks = (length + kChunk - 1) / kChunk;
    const auto chunk_of = [&](int c) { return reverse ? chunks - 1 - c : c; };
    const auto tokens_of = [&](int c) { return min(kChunk, length - chunk_of(c) * kChunk); };
    bool ok = true;

    if (warp == kIssueWarp)
    {
        // The whole warp walks the loop; only the products and copies themselves are one lane's, by predicate and not by a branch, so
        // that addresses and descriptors stay in uniform registers (a product costs 30 to 60 cycles of issue less than with a branch).
        const int hq = head / p.q.group, hk = head / p.k.group, hv = head / p.v.group, n = a.offsets == nullptr ? static_cast<int>(item.sequence) : 0;
        const uint32_t leader = elect_lane();
        const auto load = [&](int c) {
            unsigned char *stage = smem + c % L::kStages * L::kStage;
            uint64_t *bar = &sh.full[c % L::kStages];
            const int t = static_cast<int>(item.begin) + chunk_of(c) * kChunk;
            if (leader)
            {
                mbar_arrive_expect_tx(bar, L::kStage);
#pragma unroll
                for (int part = 0; part < IN; ++part)
                {
                    const int at = n + part * maps.sequences;
#pragma unroll
                    for (int i = 0; i < NQ; ++i)
                    {
                        box_load(stage + L::kQ + (part * NQ + i) * kBox, &maps.q[pass], i * kBoxColumns, hq, t, at, bar);
                        box_load(stage + L::kK + (part * NQ + i) * kBox, &maps.k[pass], i * kBoxColumns, hk, t, at, bar);
                    }
#pragma unroll
                    for (int i = 0; i < NV; ++i) box_load(stage + L::kV + (part * NV + i) * kBox, &maps.v[pass], i * kBoxColumns, hv, t, at, bar);
                }
            }
            __syncwarp();
        };
        int loaded = 0;
        for (; loaded < min(chunks, L::kStages > 1 ? L::kStages - 1 : 1); ++loaded) load(loaded);
        const uint32_t base = smem_addr(smem);
        constexpr uint32_t by_columns = umma_shape(kChunk, false, false), near_shape = umma_shape(kChunk, true, false),
                           change_shape = umma_shape(NQ * 64, true, true);
        const uint64_t scaled = umma_operand(base + L::kScaled, kBox, 1024), weights = umma_operand(base + L::kWeights, 16, 1024);
        // descriptors count in units of 16 bytes
        const auto issue_scores = [&](int c) {
            const uint32_t stage = base + c % L::kStages * L::kStage;
            const uint64_t q = umma_operand(stage + L::kQ, 16, 1024), k = umma_operand(stage + L::kK, 16, 1024);
            for_pairs<IN, IN>([&](int x, int y, bool later) {
#pragma unroll
                for (int i = 0; i < NQ * 4; ++i)
                    umma(leader, kScores, q + (x * NQ * kBox + i / 4 * kBox + i % 4 * 32) / 16, k + (y * NQ * kBox + i / 4 * kBox + i % 4 * 32) / 16, by_columns,
                         later || i > 0);
            });
            umma_commit(leader, &sh.scores);
        };
        int c = 0;
        if (chunks > 0)
        {
            ok = all_wait(&sh.full[0], 0);
            if (ok) issue_scores(0);
        }
#pragma unroll 1
        for (; c < chunks && ok; ++c)
        {
            const uint32_t stage = base + c % L::kStages * L::kStage, parity = c & 1;
            const uint64_t q = umma_operand(stage + L::kQ, 16, 1024), v = umma_operand(stage + L::kV, NV == 2 ? kBox : 0, 1024);
            // `ready` comes after `full`
            ok = (c == 0 || all_wait(&sh.change_free, parity ^ 1)) && all_wait(&sh.ready[c % L::kStages], c / L::kStages & 1);
            if (!ok) break;
            tmem_fence_after_sync();
            for_pairs<IN, 3>([&](int x, int y, bool later) {
#pragma unroll
                for (int k = 0; k < kChunk / 16; ++k)
                    umma(leader, kDelta, v + (x * NV * kBox + k * 2048) / 16, scaled + (y * NQ * kBox + k * 2048) / 16, change_shape, later || k > 0);
            });
            umma_commit(leader, &sh.change);
            // the previous chunk's results have been read, and before that its end state was published
            ok = c == 0 ? all_wait(&sh.state, 0) : all_wait(&sh.out_free, parity ^ 1);
            if (!ok) break;
            tmem_fence_after_sync();
            for_pairs<SP, IN>([&](int x, int y, bool later) {
#pragma unroll
                for (int i = 0; i < NQ * 4; ++i)
                    umma_tmem(leader, kFar, L::kState + x * NQ * 32 + i * 8, q + (y * NQ * kBox + i / 4 * kBox + i % 4 * 32) / 16, by_columns,
                              later || i > 0);
            });
            // all of the previous chunk's products were waited for by the readers of their results: its stage is free
            if (L::kStages > 1 && loaded < chunks) load(loaded++);
            ok = all_wait(&sh.weights, parity);
            if (!ok) break;
            tmem_fence_after_sync();
            for_pairs<IN, SP>([&](int x, int y, bool later) {
#pragma unroll
                for (int k = 0; k < kChunk / 16; ++k)
                    umma(leader, kNear, v + (x * NV * kBox + k * 2048) / 16, weights + (y * kBox + k * 32) / 16, near_shape, later || k > 0);
            });
            umma_commit(leader, &sh.out);
            if (L::kStages == 1 && loaded < chunks)
            {
                // the only stage: free when this chunk's results have been read
                ok = all_wait(&sh.out_free, parity);
                if (!ok) break;
                load(loaded++);
            }
            if (c + 1 < chunks)
            {
                ok = all_wait(&sh.full[(c + 1) % L::kStages], (c + 1) / L::kStages & 1);
                if (!ok) break;
                issue_scores(c + 1);
            }
        }
        // no product is in flight when this warp gives its tensor memory back
        if (ok && chunks > 0) ok = all_wait(&sh.out, (chunks - 1) & 1);
        if (!ok)
        {
            if (lane == 0) *a.wait_flag = 1;
            // copies and products of this CTA that are still in flight
            for (int i = c; i < loaded; ++i) all_wait(&sh.full[i % L::kStages], i / L::kStages & 1);
            umma_commit(leader, &sh.drained);
            all_wait(&sh.drained, 0);
        }
    }
    else if (warp >= kStateWarps)
    {
        const bool scores = warp % 4 < 2;
        const int half = (warp - kStateWarps) / 4;
        const int id = half * 64 + warp % 2 * 32 + lane;        // among the 128 threads of either kind
        for (int c = 0; c < chunks; ++c)
        {
            unsigned char *stage = smem + c % L::kStages * L::kStage;
            const uint32_t parity = c & 1;
            const int m = tokens_of(c);
            ok = all_wait(&sh.full[c % L::kStages], c / L::kStages & 1);
            if (!ok) break;
            if (!scores)
            {
                // the three parts are read by the previous chunk's products until its change is complete
                if (c > 0) ok = all_wait(&sh.change, parity ^ 1);
                if (!ok) break;
#pragma unroll 1
                for (int i = 0; i < NQ * 4; ++i)
                {
                    const int piece = i * 128 + id, r = piece / 8 % kChunk;
                    Two y[4];
#pragma unroll
                    for (int k = IN - 1; k >= 0; --k)
                    {
                        uint4 x = *reinterpret_cast<const uint4 *>(stage + L::kK + k * NQ * kBox + piece * 16);
                        if (r >= m) x = make_uint4(0, 0, 0, 0);     // whatever stands behind the last token
                        const uint32_t in[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) y[j] = k == IN - 1 ? unpack_bf16(in[j]) : add2(y[j], unpack_bf16(in[j]));
                    }
                    const float w = sh.left[r >= m ? 0 : reverse ? r + 1 : m - 1 - r];
                    uint32_t part[3][4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                    {
                        y[j] = mul2(y[j], two(w, w));
                        part[0][j] = take_part(y[j]);
                        part[1][j] = take_part(y[j]);
                        part[2][j] = pack_bf16(y[j]);
                    }
#pragma unroll
                    for (int k = 0; k < 3; ++k)
                        *reinterpret_cast<uint4 *>(smem + L::kScaled + k * NQ * kBox + piece * 16) = make_uint4(part[k][0], part[k][1], part[k][2], part[k][3]);
                }
                fence_proxy_async();
                warp_arrive(&sh.ready[c % L::kStages]);
                continue;
            }
            // Rows of V behind the last token become zeros.  So do its infinities and NaN, because a masked weight times one of them would
            // be NaN: where there are any, the rows and states that they do meet get them from the state warps.
            if (id == 0) sh.odd[(c + kRing / 2) % kRing] = 0;
            uint32_t largest = 0;           // of the magnitudes' bits, in either half
#pragma unroll 2
            for (int i = 0; i < NV * 4; ++i)
            {
                const int piece = i * 128 + id;
                uint4 *at = reinterpret_cast<uint4 *>(stage + L::kV + piece * 16);
                if (piece / 8 % kChunk >= m)
                {
#pragma unroll
                    for (int k = 0; k < IN; ++k) at[k * NV * kBox / 16] = make_uint4(0, 0, 0, 0);
                }
                const uint4 x = *at;            // the first part tells
                largest = __vmaxu2(largest, __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu)));
            }
            const bool odd = odd_pair(largest);
            if (__builtin_expect(odd, 0))
            {
#pragma unroll 1
                for (int i = 0; i < NV * 4; ++i)
                {
                    uint4 *at = reinterpret_cast<uint4 *>(stage + L::kV + (i * 128 + id) * 16);
                    const uint4 x = *at;
                    *at = make_uint4(finite_pair(x.x), finite_pair(x.y), finite_pair(x.z), finite_pair(x.w));
                }
            }
            if (odd) sh.odd[c % kRing] = 1;
            fence_proxy_async();
            warp_arrive(&sh.ready[c % L::kStages]);        // one barrier per stage: these warps may be a few chunks ahead
            // the previous chunk's weights have been read when its results have
            ok = all_wait(&sh.scores, parity) && (c == 0 || all_wait(&sh.out_free, parity ^ 1));
            if (!ok) break;
            tmem_fence_after_sync();
            const int r = warp % 4 * 32 + lane;
            const unsigned first = reverse ? r : 0, seen = reverse ? m - 1 - r : r;     // columns first .. first + seen
            const bool none = reverse && r >= m;
            // one of the four warps holds a block that no row sees: its zeros stay from the first chunk
            const bool blank = c > 0 && (reverse ? half * 32 < warp % 4 * 32 : half * 32 > warp % 4 * 32);
#pragma unroll 1
            for (int i = half * 4; i < half * 4 + 4 && !blank; ++i)
            {
                uint32_t x[8], part[SP][4];
                tmem_load_8(tmem + kScores + (static_cast<uint32_t>(warp % 4 * 32) << 16) + i * 8, x);
                const float *weight = sh.weight + kChunk - r + i * 8;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    // not a product with a zero: the score may be an infinity or NaN of another token
                    const uint32_t y0 = i * 8 + 2 * j - first > seen ? 0u : x[2 * j], y1 = i * 8 + 2 * j + 1 - first > seen ? 0u : x[2 * j + 1];
                    Two z = mul2(two(y0, y1), two(weight[2 * j], weight[2 * j + 1]));
#pragma unroll
                    for (int k = 0; k < SP - 1; ++k) part[k][j] = take_part(z);
                    part[SP - 1][j] = pack_bf16(z);
                }
                unsigned char *to = smem + L::kWeights + r * 128 + (i ^ (r & 7)) * 16;
#pragma unroll
                for (int k = 0; k < SP; ++k)
                    *reinterpret_cast<uint4 *>(to + k * kBox) = none ? make_uint4(0, 0, 0, 0) : make_uint4(part[k][0], part[k][1], part[k][2], part[k][3]);
            }
            tmem_fence_before_sync();
            fence_proxy_async();
            warp_arrive(&sh.weights);
        }
        if (!ok && lane == 0) *a.wait_flag = 1;
    }
    else
    {
        // this thread's row of the transposed state, and which quarter of its columns
        const int b = warp % 4 * 32 + lane, part = warp / 4, d0 = part * PART, r0 = part * 16;
        const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
        const bool used = b < p.dv;
        Two s[PART / 2];
        const int64_t size = static_cast<int64_t>(p.dq) * p.dv;
        {
            const float *from = nullptr;
            int turned = 0;
            if (cut) from = static_cast<const float *>(p.segment_states) + (item.segment_state * a.heads + head) * size;
            else if (p.initial != nullptr)
            {
                from = static_cast<const float *>(p.initial) + (item.state * a.heads + head) * size;
                turned = p.turned;
            }
            // one address for all of them, so that the loads go out together
            const int along = turned ? 1 : p.dv, mine = turned ? b * p.dq : b;
            const int there = from != nullptr && used ? min(PART, p.dq - d0) : 0;
            float x[PART];
#pragma unroll
            for (int j = 0; j < PART; ++j) x[j] = j < there ? from[mine + (d0 + j) * along] : 0.0f;
#pragma unroll
            for (int j = 0; j < PART; j += 2) s[j / 2] = two(x[j], x[j + 1]);
        }
        const auto publish = [&]() {
            // the state as the A operand of the next chunk: bf16 parts, pairs of columns
#pragma unroll
            for (int j = 0; j < PART; j += 16)
            {
                uint32_t part[SP][8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                {
                    Two x = s[j / 2 + i];
#pragma unroll
                    for (int k = 0; k < SP - 1; ++k) part[k][i] = take_part(x);
                    part[SP - 1][i] = pack_bf16(x);
                }
#pragma unroll
                for (int k = 0; k < SP; ++k) tmem_store_8(tmem + L::kState + k * NQ * 32 + lanes + (d0 + j) / 2, part[k]);
            }
            tmem_wait_stores();
        };
        publish();
        tmem_fence_before_sync();
        warp_arrive(&sh.state);
        // rows of `out` are a 32-bit number of bytes apart
        const uint32_t step = static_cast<uint32_t>(p.out.token) * static_cast<uint32_t>(sizeof(OUT));
        char *out = reinterpret_cast<char *>(rows_of<OUT>(p.out, a, item.sequence, head) + item.begin * p.out.token + b);
        float keep = 1, rest = 0;
        int kept = 0;
        for (int c = 0; c < chunks; ++c)
        {
            const uint32_t parity = c & 1;
            const int m = tokens_of(c);
            if (m != kept)
            {
                // what is left of the state after m tokens, to twice the digits: the rounding of one factor would come back in every chunk
                const double exact = exp(g * m);
                keep = static_cast<float>(exact);
                rest = static_cast<float>(exact - static_cast<double>(keep));
                kept = m;
            }
            ok = all_wait(&sh.change, parity);
            if (!ok) break;
            tmem_fence_after_sync();
            const Two keeps = two(keep, keep), rests = two(rest, rest);
#pragma unroll
            for (int j = 0; j < PART; j += 16)
            {
                uint32_t x[16];
                tmem_load_16(tmem + kDelta + lanes + d0 + j, x);
#pragma unroll
                for (int i = 0; i < 16; i += 2) s[(j + i) / 2] = fma2(keeps, s[(j + i) / 2], fma2(rests, s[(j + i) / 2], two(x[i], x[i + 1])));
            }
            tmem_fence_before_sync();
            warp_arrive(&sh.change_free);
            // A column of V with an infinity or NaN: the state's, and the rows' that see its token, become NaN.  `odd`: the first such
            // token in the order of time, as a row.
            int odd = reverse ? -1 : kChunk;
            if (__builtin_expect(sh.odd[c % kRing] != 0, 0) && used)
            {
                const __nv_bfloat16 *v = rows_of<const __nv_bfloat16>(p.v, a, item.sequence, head) + (item.begin + chunk_of(c) * kChunk) * p.v.token + b;
#pragma unroll 1
                for (int t = 0; t < m; ++t)
                    if (!isfinite(__bfloat162float(v[t * p.v.token]))) odd = reverse ? t : min(odd, t);
                if (odd >= 0 && odd < kChunk)
#pragma unroll
                    for (int j = 0; j < PART / 2; ++j) s[j] = ~0ull;
            }
            ok = all_wait(&sh.out, parity);         // the old state has been read, too
            if (!ok) break;
            tmem_fence_after_sync();
            publish();
            const float *come = sh.come[m < kChunk] + r0;
            char *row = out + static_cast<int64_t>(chunk_of(c) * kChunk + r0) * step;
#pragma unroll
            for (int h = 0; h < 16; h += 8)
            {
                uint32_t near[8], far[8];
                tmem_load_8(tmem + kNear + lanes + r0 + h, near);
                tmem_load_8(tmem + kFar + lanes + r0 + h, far);
                if (h == 8)
                {
                    tmem_fence_before_sync();
                    warp_arrive(&sh.out_free);
                }
                if (__builtin_expect(odd >= 0 && odd < kChunk, 0))
                {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (reverse ? r0 + h + i <= odd : r0 + h + i >= odd) near[i] = 0x7fffffffu;
                }
                const int rows = used ? m - r0 - h : 0;
                const auto write = [&](bool whole) {
#pragma unroll
                    for (int i = 0; i < 8; i += 2)
                    {
                        const Two o = fma2(*reinterpret_cast<const Two *>(come + h + i), two(far[i], far[i + 1]), two(near[i], near[i + 1]));
                        char *to = row + static_cast<uint64_t>(step) * (h + i), *after = row + static_cast<uint64_t>(step) * (h + i + 1);
                        put_two(reinterpret_cast<OUT *>(to), reinterpret_cast<OUT *>(after), o, whole || i < rows, whole || i + 1 < rows);
                    }
                };
                if (rows >= 8) write(true);
                else if (rows > 0) write(false);
            }
        }
        if (!ok && lane == 0) *a.wait_flag = 1;
        float *to = nullptr;
        int turned = 0;
        if (item.last && p.final != nullptr)
        {
            to = static_cast<float *>(p.final) + (item.state * a.heads + head) * size;
            turned = p.turned;
        }
        if (to != nullptr && used)
        {
            const int along = turned ? 1 : p.dv, mine = turned ? b * p.dq : b;
#pragma unroll
            for (int j = 0; j < PART; ++j)
                if (d0 + j < p.dq) to[mine + (d0 + j) * along] = j % 2 ? second_of(s[j / 2]) : first_of(s[j / 2]);
        }
    }
    tmem_fence_before_sync();
    __syncthreads();
    if (warp == kIssueWarp) tmem_free(sh.tmem, kColumns);
}

// The state that a segment alone would end with: the sum over its tokens of what is left of k v^T at its end.  The weights reach to the
// segment's end, so no state has to decay: the chunks are walked away from that end with a running factor.  16 warps make K~ (two
// buffers) and add up the chunks' products (two accumulators); one issues.
template <int NQ, int NV, int IN>
struct StateLayout
{
    static constexpr int kWarps = 17, kBlock = kWarps * 32, kMakers = 512;
    static constexpr int kParts = 3 * NQ * kBox;                // K~
    static constexpr int kK = 0, kV = IN * NQ * kBox, kStage = IN * (NQ + NV) * kBox;
    static constexpr int kFits = (kSmem - 2 * kParts - 3072) / kStage, kStages = kFits < (NQ == 2 ? 3 : 4) ? kFits : NQ == 2 ? 3 : 4;
    static constexpr int kScaled = kStages * kStage;
    static constexpr int kTables = kScaled + 2 * kParts;
    static constexpr int kDynamic = kTables + 1024 + 1024;
    static constexpr uint32_t kColumns = NQ * 128;             // two accumulators
};

struct StateShared
{
    float left[kChunk + 4];
    uint32_t tmem;
    uint64_t full[4], ready[2], done[2], drained;
};

template <int NQ, int NV, int IN>
__global__ void __launch_bounds__(StateLayout<NQ, NV, IN>::kBlock, 1) attention_states_kernel(const __grid_constant__ AttentionArgs a, const __grid_constant__ Maps maps)
{
    using L = StateLayout<NQ, NV, IN>;
    const int pass = blockIdx.y;
    const AttentionPass &p = a.pass[pass];
    const int head = blockIdx.x % a.heads;
    const int64_t item_index = blockIdx.x / a.heads;
    const bool reverse = p.reverse != 0;
    const SegmentItem item = find_item(a, item_index, reverse);
    if (item.sequence < 0 || item.last || segments_of(item.sequence_end - item.sequence_begin, a.segment) == 1) return;

    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    StateShared &sh = *reinterpret_cast<StateShared *>(smem + L::kTables);
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x / 32), 0), lane = threadIdx.x % 32;
    const double g = decay_log<float>(a.log_decay, head);
    if (threadIdx.x <= kChunk) sh.left[threadIdx.x] = static_cast<float>(exp(g * threadIdx.x) * p.state_scale);
    if (threadIdx.x == 0)
    {
        for (int i = 0; i < L::kStages; ++i) mbar_init(&sh.full[i], 1);
        for (int i = 0; i < 2; ++i)
        {
            mbar_init(&sh.ready[i], L::kMakers / 32);
            mbar_init(&sh.done[i], 1);
        }
        mbar_init(&sh.drained, 1);
        fence_mbar_init();
    }
    if (warp == 16) tmem_alloc(&sh.tmem, L::kColumns);
    tmem_fence_before_sync();
    __syncthreads();
    tmem_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
    const int length = static_cast<int>(item.end - item.begin), chunks = (length + kChunk - 1) / kChunk;
    const auto chunk_of = [&](int c) { return reverse ? c : chunks - 1 - c; };      // away from the end, in time
    bool ok = true;

    if (warp == 16)
    {
        const int hk = head / p.k.group, hv = head / p.v.group, n = a.offsets == nullptr ? static_cast<int>(item.sequence) : 0;
        const uint32_t leader = elect_lane(), base = smem_addr(smem);
        const auto load = [&](int c) {
            unsigned char *stage = smem + c % L::kStages * L::kStage;
            uint64_t *bar = &sh.full[c % L::kStages];
            const int t = static_cast<int>(item.begin) + chunk_of(c) * kChunk;
            if (leader)
            {
                mbar_arrive_expect_tx(bar, L::kStage);
#pragma unroll
                for (int part = 0; part < IN; ++part)
                {
                    const int at = n + part * maps.sequences;
#pragma unroll
                    for (int i = 0; i < NQ; ++i) box_load(stage + L::kK + (part * NQ + i) * kBox, &maps.k[pass], i * kBoxColumns, hk, t, at, bar);
#pragma unroll
                    for (int i = 0; i < NV; ++i) box_load(stage + L::kV + (part * NV + i) * kBox, &maps.v[pass], i * kBoxColumns, hv, t, at, bar);
                }
            }
            __syncwarp();
        };
        int loaded = 0, c = 0;
        for (; loaded < min(chunks, L::kStages > 1 ? L::kStages - 1 : 1); ++loaded) load(loaded);
        constexpr uint32_t shape = umma_shape(NQ * 64, true, true);
#pragma unroll 1
        for (; c < chunks; ++c)
        {
            ok = all_wait(&sh.ready[c & 1], c / 2 & 1);
            if (!ok) break;
            tmem_fence_after_sync();
            const uint64_t v = umma_operand(base + c % L::kStages * L::kStage + L::kV, NV == 2 ? kBox : 0, 1024),
                           k = umma_operand(base + L::kScaled + (c & 1) * L::kParts, kBox, 1024);
            for_pairs<IN, 3>([&](int x, int y, bool later) {
#pragma unroll
                for (int i = 0; i < kChunk / 16; ++i)
                    umma(leader, tmem + (c & 1) * NQ * 64, v + (x * NV * kBox + i * 2048) / 16, k + (y * NQ * kBox + i * 2048) / 16, shape, later || i > 0);
            });
            umma_commit(leader, &sh.done[c & 1]);
            if (loaded < chunks)
            {
                // into the previous chunk's stage (this one's, where there is one stage)
                const int freed = L::kStages > 1 ? c - 1 : c;
                if (freed >= 0) ok = all_wait(&sh.done[freed & 1], freed / 2 & 1);
                if (!ok) break;
                load(loaded++);
            }
        }
        if (ok) ok = all_wait(&sh.done[(chunks - 1) & 1], (chunks - 1) / 2 & 1);
        if (!ok)
        {
            if (lane == 0) *a.wait_flag = 1;
            // copies and products of this CTA that are still in flight
            for (int i = c; i < loaded; ++i) all_wait(&sh.full[i % L::kStages], i / L::kStages & 1);
            umma_commit(leader, &sh.drained);
            all_wait(&sh.drained, 0);
        }
    }
    else
    {
        const double whole = exp(g * kChunk);
        double factor = 1;
        const int b = warp % 4 * 32 + lane, d0 = warp / 4 * NQ * 16;
        Two sum[NQ * 8];
#pragma unroll
        for (int j = 0; j < NQ * 8; ++j) sum[j] = two(0.0f, 0.0f);
        const auto add = [&](int c) {
#pragma unroll
            for (int j = 0; j < NQ * 16; j += 16)
            {
                uint32_t x[16];
                tmem_load_16(tmem + (static_cast<uint32_t>(warp % 4 * 32) << 16) + (c & 1) * NQ * 64 + d0 + j, x);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[j / 2 + i] = add2(sum[j / 2 + i], two(x[2 * i], x[2 * i + 1]));
            }
            tmem_fence_before_sync();
        };
        for (int c = 0; c < chunks; ++c)
        {
            unsigned char *stage = smem + c % L::kStages * L::kStage, *scaled = smem + L::kScaled + (c & 1) * L::kParts;
            const int m = min(kChunk, length - chunk_of(c) * kChunk);
            // the buffer of K~ that this chunk takes was read by the products that were added up last
            ok = all_wait(&sh.full[c % L::kStages], c / L::kStages & 1);
            if (!ok) break;
            const float f = static_cast<float>(factor);
#pragma unroll
            for (int i = 0; i < NQ; ++i)
            {
                const int piece = i * L::kMakers + threadIdx.x, r = piece / 8 % kChunk;
                Two y[4];
#pragma unroll
                for (int k = IN - 1; k >= 0; --k)
                {
                    uint4 x = *reinterpret_cast<const uint4 *>(stage + L::kK + k * NQ * kBox + piece * 16);
                    if (r >= m) x = make_uint4(0, 0, 0, 0);
                    const uint32_t in[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[j] = k == IN - 1 ? unpack_bf16(in[j]) : add2(y[j], unpack_bf16(in[j]));
                }
                const float w = sh.left[r >= m ? 0 : reverse ? r + 1 : m - 1 - r] * f;
                uint32_t part[3][4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    y[j] = mul2(y[j], two(w, w));
                    part[0][j] = take_part(y[j]);
                    part[1][j] = take_part(y[j]);
                    part[2][j] = pack_bf16(y[j]);
                }
#pragma unroll
                for (int k = 0; k < 3; ++k)
                    *reinterpret_cast<uint4 *>(scaled + k * NQ * kBox + piece * 16) = make_uint4(part[k][0], part[k][1], part[k][2], part[k][3]);
            }
            if (m < kChunk)
            {
#pragma unroll
                for (int i = 0; i < NV; ++i)
                {
                    const int piece = i * L::kMakers + threadIdx.x;
                    if (piece / 8 % kChunk >= m)
#pragma unroll
                        for (int k = 0; k < IN; ++k) *reinterpret_cast<uint4 *>(stage + L::kV + k * NV * kBox + piece * 16) = make_uint4(0, 0, 0, 0);
                }
            }
            fence_proxy_async();
            warp_arrive(&sh.ready[c & 1]);
            factor *= m == kChunk ? whole : exp(g * m);
            if (c == 0) continue;
            ok = all_wait(&sh.done[(c - 1) & 1], (c - 1) / 2 & 1);
            if (!ok) break;
            tmem_fence_after_sync();
            add(c - 1);
        }
        if (ok) ok = all_wait(&sh.done[(chunks - 1) & 1], (chunks - 1) / 2 & 1);
        if (ok)
        {
            tmem_fence_after_sync();
            add(chunks - 1);
            float *to = static_cast<float *>(p.segment_states) + (item.segment_state * a.heads + head) * (static_cast<int64_t>(p.dq) * p.dv);
#pragma unroll
            for (int j = 0; j < NQ * 16; ++j)
                if (b < p.dv && d0 + j < p.dq) to[(d0 + j) * p.dv + b] = j % 2 ? second_of(sum[j / 2]) : first_of(sum[j / 2]);
        }
        else if (lane == 0) *a.wait_flag = 1;
    }
    tmem_fence_before_sync();
    __syncthreads();
    if (warp == 16) tmem_free(tmem, L::kColumns);
}

template <int NQ, int NV, int IN, class OUT>
int launch_as(const AttentionArgs &a, const Maps &maps, cudaStream_t stream)
{
    using L = Layout<NQ, NV, IN>;
    const char *name = "acro_b200_linear_attention";
    cudaError_t status = allow_dynamic_smem(attention_mma_kernel<NQ, NV, IN, OUT>, L::kDynamic);
    if (status != cudaSuccess) return fail_cuda(status, name);
    const dim3 grid(static_cast<unsigned>(a.items * a.heads), a.passes);
    attention_mma_kernel<NQ, NV, IN, OUT><<<grid, kBlock, L::kDynamic, stream>>>(a, maps);
    return launch_status(name);
}

// T: the type of results that are not sums.
template <int NQ, int NV, int IN, class T>
int launch(const AttentionArgs &a, const Maps &maps, bool states_only, cudaStream_t stream)
{
    if (states_only)
    {
        using L = StateLayout<NQ, NV, IN>;
        const char *name = "acro_b200_linear_attention";
        cudaError_t status = allow_dynamic_smem(attention_states_kernel<NQ, NV, IN>, L::kDynamic);
        if (status != cudaSuccess) return fail_cuda(status, name);
        const dim3 grid(static_cast<unsigned>(a.items * a.heads), a.passes);
        attention_states_kernel<NQ, NV, IN><<<grid, L::kBlock, L::kDynamic, stream>>>(a, maps);
        return launch_status(name);
    }
    // one launch per kind of output: passes of the gradient write rows of sums when key and value heads are shared
    int status = ACRO_B200_OK;
    AttentionArgs part = a;
    Maps of = maps;
    for (int first = 0; first < a.passes && status == ACRO_B200_OK; first += part.passes)
    {
        part.passes = 0;
        while (first + part.passes < a.passes && (std::is_same<T, float>::value || a.pass[first + part.passes].sums == a.pass[first].sums))
        {
            part.pass[part.passes] = a.pass[first + part.passes];
            of.q[part.passes] = maps.q[first + part.passes];
            of.k[part.passes] = maps.k[first + part.passes];
            of.v[part.passes] = maps.v[first + part.passes];
            ++part.passes;
        }
        status = a.pass[first].sums ? launch_as<NQ, NV, IN, float>(part, of, stream) : launch_as<NQ, NV, IN, T>(part, of, stream);
    }
    return status;
}

template <int IN, class T>
int launch_parts(const AttentionArgs &a, const Maps &maps, int q, int v, bool states_only, cudaStream_t stream)
{
    if (q == 1) return v == 1 ? launch<1, 1, IN, T>(a, maps, states_only, stream) : launch<1, 2, IN, T>(a, maps, states_only, stream);
    return v == 1 ? launch<2, 1, IN, T>(a, maps, states_only, stream) : launch<2, 2, IN, T>(a, maps, states_only, stream);
}

}

namespace acro_b200_detail
{

// `maps` is a Maps: launches of inputs of one, two and three parts, each in a file of its own.
int attention_mma_bf16(const AttentionArgs &a, const void *maps, int q, int v, bool states_only, cudaStream_t stream);
int attention_mma_f16(const AttentionArgs &a, const void *maps, int q, int v, bool states_only, cudaStream_t stream);
int attention_mma_f32(const AttentionArgs &a, const void *maps, int q, int v, bool states_only, cudaStream_t stream);

}

#endif
