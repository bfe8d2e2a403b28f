// Linear attention with a decay for each head: what its kernels share.
//
// Per sequence and head, with lam = exp(log_decay):   S_t = lam S_(t-1) + k_t v_t^T,   o_t = scale q_t^T S_t.
// A chunk of m tokens starting from the state S (row r of the chunk, natural order):
//   o_r = scale ( come_r q_r^T S + sum_(s <= r) lam^(r-s) (q_r.k_s) v_s ),   come_r = lam^(r+1)
//   S'  = lam^m S + sum_s left_s k_s v_s^T,                                  left_s = lam^(m-1-s)
// Every gradient is a pass of the same form with its operands in other places:
//   dq = pass(q := do, k := v, v := k), forward in time, with the transposed state
//   dk = pass(q := v, k := do, v := q), dv = pass(q := k, k := q, v := do), both backward in time with the gradient of the state,
//        which a backward pass holds already decayed: sums over s >= r, come_r = lam^(m-1-r), left_s = lam^(s+1)
// so come and left change places, and the state after the first token is the gradient of the initial state.
//
// A long sequence is cut into segments so that few heads still fill the GPU: a first pass over all segments but the last
// makes each one's own state from zero, a small kernel turns these into the states the segments start from, and the main pass
// runs the segments beside one another.  That reads k and v twice, so it is done only when sequences x heads leave SMs idle.
#ifndef ACRO_B200_KERNELS_LINEAR_ATTENTION_CUH
#define ACRO_B200_KERNELS_LINEAR_ATTENTION_CUH

#include "element.cuh"

namespace acro_b200_detail
{

// Rows of one operand: element (sequence n, token t, head h, column c) at data[n * sequence + t * token + h * head + c]; with
// packed sequences `sequence` is not used and t counts over all rows.  group: query heads that share a head of this operand.
struct TokenRows
{
    void *data;
    int64_t sequence, token, head;
    int32_t group;
};

// One pass over all sequences and heads.
struct AttentionPass
{
    TokenRows q, k, v, out;
    int32_t dq, dv;                     // columns of q and k; of v and out
    int32_t reverse;                    // backward in time
    int32_t turned;                     // the user's states are [dv][dq]: read and written transposed
    int32_t packs;                      // q, k and v can be read in packs of 16 bytes of sums (set by the launch)
    int32_t sums;                       // out is in the type of sums (one row per query head, to be added up), not the element type
    double state_scale, out_scale;      // on k v^T as it enters the state, on q^T S; their product on (q.k) v
    const void *initial;                // state a sequence starts from, or null: zero
    void *final;                        // state it ends with, or null
    void *segment_states;               // [states_of_segments][heads][dq][dv], or null when no sequence is cut
};

struct AttentionArgs
{
    AttentionPass pass[3];
    int32_t passes;
    int32_t heads;
    const void *log_decay;
    const int64_t *offsets;             // sequences + 1 row numbers, or null: all sequences have `tokens` tokens
    const int32_t *slots;               // state of each sequence, or null: the n-th
    int64_t state_count;                // number of states behind `slots`
    int64_t sequences, tokens;          // tokens: with offsets, the number of rows
    int64_t segment;                    // tokens of a segment, a multiple of every kernel's chunk
    int64_t items;                      // upper bound of the number of segments of all sequences
    int *bad_index;
    int *wait_flag;
};

struct SegmentItem
{
    int64_t begin, end;                 // tokens of the sequence (of all rows when packed)
    int64_t sequence;                   // -1: no such item, or a sequence that is not there
    int64_t segment_state;              // where the states of a cut sequence's segment are kept
    int64_t sequence_begin, sequence_end;
    int64_t state;                      // which of the user's states
    int32_t last;                       // is this the sequence's last item in the order of time?
    int32_t first;
};

__host__ __device__ __forceinline__ int64_t segments_of(int64_t length, int64_t segment) { return length <= segment ? 1 : (length + segment - 1) / segment; }

// Where the state of segment `index` of a cut sequence is kept.  Packed: two places for every `segment` rows, the second for a
// sequence's first segment.  Two segments that start within the same `segment` rows are the last one of a sequence and the first one
// of the next that is cut, so that is enough, and the memory does not grow with the number of sequences.
__host__ __device__ __forceinline__ int64_t states_of_segments(int64_t sequences, int64_t tokens, int64_t segment, bool packed)
{
    return packed ? 2 * (tokens / segment + 1) : sequences * segments_of(tokens, segment);
}

__device__ __forceinline__ int64_t segment_state(const AttentionArgs &a, int64_t sequence, int64_t sequence_begin, int64_t index)
{
    if (a.offsets != nullptr) return 2 * (sequence_begin / a.segment + index) + (index == 0);
    return sequence * segments_of(a.tokens, a.segment) + index;
}

// An entry of `offsets` is bad when it is not in 0 .. rows or lower than one in front of it.  A sequence that starts or ends at a bad
// entry is skipped (and reported), so that the others have rows, and places for segments' states, of their own.

// Are all entries good?  Every thread of the CTA calls it; holds a CTA barrier.
__device__ __forceinline__ bool offsets_ascend(const int64_t *offsets, int64_t sequences, int64_t rows)
{
    bool bad = false;
    for (int64_t n = threadIdx.x; n < sequences; n += blockDim.x) bad |= offsets[n] < 0 || offsets[n + 1] < offsets[n] || offsets[n + 1] > rows;
    return __syncthreads_or(bad) == 0;
}

// Rows begin .. end-1 of sequence n, or false for one that is skipped.  `highest`: the highest entry in front of n.
__device__ __forceinline__ bool rows_of_sequence(const int64_t *offsets, int64_t n, int64_t rows, int64_t highest, int64_t &begin, int64_t &end)
{
    begin = offsets[n];
    end = offsets[n + 1];
    return begin >= 0 && begin >= highest && end >= begin && end <= rows;
}

// Which state belongs to entry n of `slots`: -1 when the entry is negative (a request that is not there), out of range or the
// same as an earlier entry (both reported).  Every thread of the CTA calls it; holds a CTA barrier.
__device__ __forceinline__ int64_t state_of(const int32_t *slots, int64_t n, int64_t count, int *bad_index)
{
    if (slots == nullptr) return n;
    const int32_t mine = slots[n];
    bool twice = false;
    if (mine >= 0)
        for (int64_t i = threadIdx.x; i < n; i += blockDim.x) twice |= slots[i] == mine;
    twice = __syncthreads_or(twice) != 0;
    if (mine < 0) return -1;
    if (twice || mine >= count)
    {
        if (threadIdx.x == 0) atomicOr(bad_index, 1);
        return -1;
    }
    return mine;
}

// Inclusive sum over the CTA's threads of two counts, before each thread's own the sums of the threads in front of it.  Every thread
// calls it; holds CTA barriers.
__device__ __forceinline__ void scan_two(int64_t &x, int64_t &y, int64_t &total_x, int64_t &total_y, int64_t (*sums)[2])
{
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
    const int64_t own_x = x, own_y = y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
    {
        const int64_t up_x = __shfl_up_sync(0xffffffffu, x, o), up_y = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o)
        {
            x += up_x;
            y += up_y;
        }
    }
    __syncthreads();
    if (lane == 31)
    {
        sums[warp][0] = x;
        sums[warp][1] = y;
    }
    __syncthreads();
    total_x = total_y = 0;
    int64_t ahead_x = 0, ahead_y = 0;
    for (int w = 0; w < warps; ++w)
    {
        if (w == warp)
        {
            ahead_x = total_x;
            ahead_y = total_y;
        }
        total_x += sums[w][0];
        total_y += sums[w][1];
    }
    x += ahead_x - own_x;
    y += ahead_y - own_y;
}

// The highest of `highest` and the `mine` of the threads in front of this one; `highest` becomes that of all threads.  Every thread calls
// it; holds CTA barriers.
__device__ __forceinline__ int64_t highest_ahead(int64_t mine, int64_t &highest, int64_t (*sums)[2])
{
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1)
    {
        const int64_t up = __shfl_up_sync(0xffffffffu, mine, o);
        if (lane >= o && up > mine) mine = up;
    }
    __syncthreads();
    if (lane == 31) sums[warp][0] = mine;
    __syncthreads();
    int64_t ahead = __shfl_up_sync(0xffffffffu, mine, 1);
    if (lane == 0 || ahead < highest) ahead = highest;
    for (int w = 0; w < warps; ++w)
    {
        if (w < warp && sums[w][0] > ahead) ahead = sums[w][0];
        if (sums[w][0] > highest) highest = sums[w][0];
    }
    return ahead;
}

// Rows of sequence base + threadIdx.x, or false.  `highest`: the highest entry in front of base, then that in front of base + blockDim.x.
// Every thread calls it; holds CTA barriers.
__device__ __forceinline__ bool next_rows(const AttentionArgs &a, int64_t base, int64_t &highest, int64_t &begin, int64_t &end, int64_t (*sums)[2])
{
    const int64_t n = base + threadIdx.x;
    const bool there = n < a.sequences;
    const int64_t ahead = highest_ahead(there ? a.offsets[n] : INT64_MIN, highest, sums);
    return there && rows_of_sequence(a.offsets, n, a.tokens, ahead, begin, end);
}

// One block of sequences in the search for item `launched`: sets found (sequence, its rows, which of its segments) if it is among them.
// `there`: thread's sequence n has the rows b .. e-1 (and is not skipped).  `before`: whole and last segments in front of the block, then
// behind it; `whole`: whole segments of all sequences.  Every thread calls it; holds CTA barriers.
__device__ __forceinline__ void find_in_block(const AttentionArgs &a, int64_t launched, int64_t n, bool there, int64_t b, int64_t e, int64_t whole,
                                              int64_t &before_last, int64_t &before_whole, int64_t *found, int64_t (*sums)[2])
{
    int64_t mine_last = 0, mine_whole = 0;
    if (there)
    {
        mine_whole = (e - b) / a.segment;
        mine_last = segments_of(e - b, a.segment) - mine_whole;
    }
    int64_t start_last = mine_last, start_whole = mine_whole, total_last, total_whole;
    scan_two(start_last, start_whole, total_last, total_whole, sums);
    start_last += before_last;
    start_whole += before_whole;
    int64_t which = -1;
    if (launched < whole && launched >= start_whole && launched < start_whole + mine_whole) which = launched - start_whole;
    if (launched >= whole && mine_last > 0 && launched - whole == start_last) which = mine_whole;
    if (which >= 0)
    {
        found[0] = n;
        found[1] = b;
        found[2] = e;
        found[3] = which;
    }
    before_last += total_last;
    before_whole += total_whole;
}

// The search among sequences of which some are skipped: their validity needs all entries in front of theirs.  A call of its own, so that the
// kernels' first instructions stay few (inlined, it cost a cold launch 3 us).
static __device__ __noinline__ void find_among_bad(const AttentionArgs &a, int64_t launched, int64_t *found, int64_t (*sums)[2])
{
    if (threadIdx.x == 0) atomicOr(a.bad_index, 1);
    int64_t all = 0, none = 0, whole, nothing, b, e, highest = INT64_MIN;
    for (int64_t base = 0; base < a.sequences; base += blockDim.x)
        if (next_rows(a, base, highest, b, e, sums)) all += (e - b) / a.segment;
    scan_two(all, none, whole, nothing, sums);
    int64_t before_last = 0, before_whole = 0;
    highest = INT64_MIN;
    for (int64_t base = 0; base < a.sequences; base += blockDim.x)
    {
        const bool there = next_rows(a, base, highest, b, e, sums);
        find_in_block(a, launched, base + threadIdx.x, there, b, e, whole, before_last, before_whole, found, sums);
    }
}

// Item `launched` of the list of all sequences' segments.  Packed sequences put their whole segments in front and their (shorter) last
// ones behind, so that the long work starts first.  Every thread of the CTA (at most 1024, whole warps) calls it and gets the same
// answer; holds CTA barriers.
__device__ __forceinline__ SegmentItem find_item(const AttentionArgs &a, int64_t launched, bool reverse)
{
    SegmentItem s;
    int64_t index;
    if (a.offsets == nullptr)
    {
        const int64_t each = segments_of(a.tokens, a.segment);
        s.sequence = launched / each;
        index = launched - s.sequence * each;
        s.sequence_begin = 0;
        s.sequence_end = a.tokens;
    }
    else
    {
        __shared__ int64_t found[4], sums[32][2];
        if (threadIdx.x == 0) found[0] = -1;
        // the number of whole segments of all sequences
        int64_t all = 0, b = 0, e = 0;
        bool bad = false;
        for (int64_t n = threadIdx.x; n < a.sequences; n += blockDim.x)
        {
            if (rows_of_sequence(a.offsets, n, a.tokens, 0, b, e)) all += (e - b) / a.segment;
            else bad = true;
        }
        if (__syncthreads_or(bad) != 0) find_among_bad(a, launched, found, sums);
        else
        {
            int64_t none = 0, whole, nothing;
            scan_two(all, none, whole, nothing, sums);
            int64_t before_last = 0, before_whole = 0;
            for (int64_t base = 0; base < a.sequences; base += blockDim.x)
            {
                const int64_t n = base + threadIdx.x;
                const bool there = n < a.sequences;
                if (there)
                {
                    b = a.offsets[n];
                    e = a.offsets[n + 1];
                }
                find_in_block(a, launched, n, there, b, e, whole, before_last, before_whole, found, sums);
            }
        }
        __syncthreads();
        s.sequence = found[0];
        s.sequence_begin = found[1];
        s.sequence_end = found[2];
        index = found[3];
    }
    if (s.sequence < 0) return s;
    s.state = state_of(a.slots, s.sequence, a.state_count, a.bad_index);
    if (s.state < 0)
    {
        s.sequence = -1;
        return s;
    }
    const int64_t count = segments_of(s.sequence_end - s.sequence_begin, a.segment);
    s.segment_state = segment_state(a, s.sequence, s.sequence_begin, index);
    s.begin = s.sequence_begin + index * a.segment;
    s.end = s.begin + a.segment < s.sequence_end ? s.begin + a.segment : s.sequence_end;
    s.first = reverse ? index == count - 1 : index == 0;
    s.last = reverse ? index == 0 : index == count - 1;
    return s;
}

template <class T>
__device__ __forceinline__ T *rows_of(const TokenRows &r, const AttentionArgs &a, int64_t sequence, int head)
{
    return static_cast<T *>(r.data) + (a.offsets == nullptr ? sequence * r.sequence : 0) + static_cast<int64_t>(head / r.group) * r.head;
}

// The logarithm of a head's decay.  A decay of zero (-inf) becomes one so small that every power but the zeroth is zero.
template <class A>
__device__ __forceinline__ A decay_log(const void *log_decay, int head)
{
    const A g = static_cast<const A *>(log_decay)[head];
    return g < A(-1e5) ? A(-1e5) : g;
}

// The pass on the tcgen05 tensor cores (linear_attention_mma.cuh).  Its inputs are bf16 rows that tiled copies can read
// (attention_mma_direct), or the planes of bf16 parts that attention_split makes of any rows of up to 32 bits, in whose place it then
// puts the planes (attention_planes_bytes for each array, one behind the other).
bool attention_mma_sizes(const AttentionArgs &a);
bool attention_mma_direct(const AttentionArgs &a);
size_t attention_planes_bytes(int type, int64_t rows, int heads, int columns);
int attention_split(AttentionArgs &a, int type, const TokenRows *arrays, const int *columns, int count, void *planes, cudaStream_t stream);
int attention_mma_launch(const AttentionArgs &a, int type, bool states_only, cudaStream_t stream);

}

#endif
