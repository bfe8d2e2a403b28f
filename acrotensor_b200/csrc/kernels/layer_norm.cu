// Layer norm of rows and its gradient.
//
//   mean = sum_f x_f / W,  rstd = 1 / sqrt(sum_f (x_f - mean)^2 / W + eps),  xhat = (x - mean) rstd,  y = xhat w + b
//   g = dy w,  dx = rstd (g - sum(g)/W - xhat sum(g xhat)/W),  dw_f = sum_rows dy xhat,  db_f = sum_rows dy
//
// Both are bound by HBM: 2 and 3 elements moved per entry against about ten operations.  So a row is read once, stays in
// registers between its moments and its result, and leaves once.  A row belongs to a group of G threads (a power of two up to a warp,
// or whole warps); a CTA holds several groups when rows are short.  Groups walk over rows and load the next row's bytes before
// they work on one.  Elements are worked on in pairs, with weight and bias in registers, and a group has a barrier of its own.
// The variance is the mean square of the centred entries (a second walk over the registers), not a difference of moments, which
// cancels for rows far from zero.
//
// 16384 x 4096 in fp32: 91 us, gradient 151 us (90 and 81 % of the measured copy rate).  In bf16 52 and 93 us (79 and 66 %; a copy of these
// arrays takes 44 us, a sum of two of them 60): half the bytes for the same instructions, so that issue (55 to 60 % of its slots) and
// the barriers' latency count, with 16 warps an SM for want of registers.  More rows on their way did not help: two or three rows
// ahead in registers 67 and 83 us, a ring of four in shared memory (bulk copies) 68 and 95 us.
//
// The gradient's column sums run over all rows: a thread owns the same columns of every row that its group takes, so the sums over
// those rows stay in its registers (in shared memory beyond 16 columns a thread); the groups of a CTA are added in ascending order, a CTA
// leaves one row of partial sums, and a second kernel adds these in ascending order.  No atomics: the same bits on every run on
// one device.
#include "element.cuh"

#include <algorithm>

using namespace acro_b200_detail;

namespace
{

constexpr int kMaxThreads = 512;       // of one group
constexpr int kWideThreads = 512;

struct NormArgs
{
    const void *x, *w, *b, *dy;
    void *y;                            // the result, or dx
    void *mean, *rstd;                  // written by the forward pass (or null), read by the gradient
    void *partial;                      // gradient: [CTAs][2][width] sums
    int64_t rows, width, x_stride, y_stride, dy_stride;
    double eps;
    int group;                          // threads of one row
};

// Sum over the threads of a row's group, each of whom calls it.  `slot`: the group's own part of shared memory, one entry per warp.  Two
// sums in a row use different slots: then everybody has read the one before the last when a barrier lets the next be written.
template <int N, class A>
__device__ __forceinline__ void group_sum(A (&v)[N], A *slot, int group)
{
    const int within = group < 32 ? group : 32;
    for (int o = within / 2; o > 0; o >>= 1)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
    const int warps = group / 32;
    if (warps <= 1) return;
    struct alignas(N * sizeof(A)) All { A v[N]; };
    All *all = reinterpret_cast<All *>(slot);
    if (threadIdx.x % 32 == 0)
    {
        All &mine = all[threadIdx.x % group / 32];
#pragma unroll
        for (int i = 0; i < N; ++i) mine.v[i] = v[i];
    }
    // the group's own barrier
    asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / group), "r"(group) : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0;
#pragma unroll 4
    for (int k = 0; k < warps; ++k)
    {
        const All other = all[k];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += other.v[i];
    }
}

// 1 / sqrt(v).  In 32 bits the function's two steps of error less a Newton step: a third of the instructions of a root and a quotient.
__device__ __forceinline__ double inverse_root(double v) { return 1.0 / sqrt(v); }
__device__ __forceinline__ float inverse_root(float v)
{
    const float r = rsqrtf(v), left = fmaf(-v * r, r, 1.0f);
    return left == left ? fmaf(0.5f * r, left, r) : r;       // zero and infinity have no step
}

// THREADS: the largest CTA (256 when rows are short enough: twice the registers a thread, and two CTAs an SM.  Left to itself the compiler took
// 152 registers in bf16 and one CTA: 66 us instead of 52 for 16384 x 4096; fp64 needs them).
template <class T, int VEC, int COLS, int THREADS>
__global__ void __launch_bounds__(THREADS, sizeof(T) < 8 ? 512 / THREADS : 1) norm_kernel(NormArgs a)
{
    using A = typename Element<T>::Acc;
    using P = typename PairOf<A>::type;
    using Row = RowPart<T, VEC, COLS>;
    __shared__ A slots[2][THREADS / 32];
    const int groups = blockDim.x / a.group, mine = threadIdx.x / a.group, lane = threadIdx.x % a.group, width = static_cast<int>(a.width);
    const int slot = mine * (a.group / 32);
    const A inv = A(1) / static_cast<A>(width);
    const int64_t step = static_cast<int64_t>(gridDim.x) * groups;
    int64_t base = static_cast<int64_t>(blockIdx.x) * groups;
    // the thread's columns of weight and bias stay in registers (one and zero where there are none)
    Row next, weight, bias;
    const A eps = static_cast<A>(a.eps);
    const T *from = static_cast<const T *>(a.x) + (base + mine) * a.x_stride;
    T *to = static_cast<T *>(a.y) + (base + mine) * a.y_stride;
    const int64_t from_step = step * a.x_stride, to_step = step * a.y_stride;
    const auto fetch = [&](int64_t row) {
        if (row < a.rows) next.load(from, lane, a.group, width);
        from += from_step;
    };
    fetch(base + mine);
    if (a.w != nullptr) weight.load(static_cast<const T *>(a.w), lane, a.group, width);
    else weight.fill(narrow2<T>(two(A(1), A(1))));
    if (a.b != nullptr) bias.load(static_cast<const T *>(a.b), lane, a.group, width);
    else bias.fill(narrow2<T>(two(A(0), A(0))));
    for (; base < a.rows; base += step)
    {
        const int64_t row = base + mine;
        const bool there = row < a.rows;
        P x[COLS / 2], sum = two(A(0), A(0));
#pragma unroll
        for (int k = 0; k < COLS / 2; ++k)
        {
            x[k] = widen2<T>(next.pair[k]);
            sum = add2(sum, x[k]);
        }
        fetch(row + step);
        A s[1] = {first_of(sum) + second_of(sum)};
        group_sum(s, slots[0] + slot, a.group);
        const A mean = s[0] * inv;
        const P means = two(mean, mean);
        sum = two(A(0), A(0));
#pragma unroll
        for (int k = 0; k < COLS / 2; ++k)
        {
            // columns behind the width weigh nothing; a pack lies before the width or behind it
            if (Row::column(k, 0, lane, a.group) >= width) continue;
            x[k] = sub2(x[k], means);
            if (VEC == 1 && Row::column(k, 1, lane, a.group) >= width) x[k] = two(first_of(x[k]), A(0));
            sum = fma2(x[k], x[k], sum);
        }
        s[0] = first_of(sum) + second_of(sum);
        group_sum(s, slots[1] + slot, a.group);
        const A rstd = inverse_root(s[0] * inv + eps);
        T *out_row = to;
        to += to_step;
        if (!there) continue;
        if (lane == 0)
        {
            if (a.mean != nullptr) static_cast<A *>(a.mean)[row] = mean;
            if (a.rstd != nullptr) static_cast<A *>(a.rstd)[row] = rstd;
        }
        const P scale = two(rstd, rstd);
        Row out;
#pragma unroll
        for (int k = 0; k < COLS / 2; ++k) out.pair[k] = narrow2<T>(fma2(mul2(x[k], scale), widen2<T>(weight.pair[k]), widen2<T>(bias.pair[k])));
        out.store(out_row, lane, a.group, width);
    }
}

// Rows wider than a group's registers hold: three walks over the row, the later two mostly from L2.
template <class T>
__global__ void __launch_bounds__(kWideThreads) norm_wide_kernel(NormArgs a)
{
    using A = typename Element<T>::Acc;
    __shared__ A slots[2][kWideThreads / 32];
    const int64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const A inv = A(1) / static_cast<A>(a.width);
    A s[1] = {0};
    for (int64_t c = threadIdx.x; c < a.width; c += kWideThreads) s[0] += widen(x[c]);
    group_sum(s, slots[0], kWideThreads);
    const A mean = s[0] * inv;
    s[0] = 0;
    for (int64_t c = threadIdx.x; c < a.width; c += kWideThreads)
    {
        const A d = widen(x[c]) - mean;
        s[0] += d * d;
    }
    group_sum(s, slots[1], kWideThreads);
    const A rstd = inverse_root(s[0] * inv + static_cast<A>(a.eps));
    if (threadIdx.x == 0)
    {
        if (a.mean != nullptr) static_cast<A *>(a.mean)[row] = mean;
        if (a.rstd != nullptr) static_cast<A *>(a.rstd)[row] = rstd;
    }
    T *y = static_cast<T *>(a.y) + row * a.y_stride;
    for (int64_t c = threadIdx.x; c < a.width; c += kWideThreads)
    {
        A v = (widen(x[c]) - mean) * rstd;
        if (a.w != nullptr) v *= widen(static_cast<const T *>(a.w)[c]);
        if (a.b != nullptr) v += widen(static_cast<const T *>(a.b)[c]);
        y[c] = narrow<T>(v);
    }
}

// Up to 16 columns a thread the column sums are registers; beyond that each thread keeps its own in shared memory (sums[2][width],
// touched by their owner alone until the end).
template <class T, int VEC, int COLS, int THREADS>
__global__ void __launch_bounds__(THREADS, sizeof(T) < 8 ? 512 / THREADS : 1) norm_gradient_kernel(NormArgs a)
{
    using A = typename Element<T>::Acc;
    using P = typename PairOf<A>::type;
    using Row = RowPart<T, VEC, COLS>;
    constexpr bool kRegisters = COLS <= 16;
    constexpr int kSums = kRegisters ? COLS / 2 : 1;
    __shared__ __align__(16) A slots[2][2 * THREADS / 32];
    extern __shared__ __align__(16) unsigned char dynamic[];
    // pair k of thread t at entry k * threads + t (dw, then db), or [groups][2][width] when groups are added up
    P *own = reinterpret_cast<P *>(dynamic);
    A *sums = reinterpret_cast<A *>(own);
    const int groups = blockDim.x / a.group, mine = threadIdx.x / a.group, lane = threadIdx.x % a.group, width = static_cast<int>(a.width);
    const int slot = mine * (a.group / 32) * 2;
    int turn = 0;
    const A inv = A(1) / static_cast<A>(width);
    P dw[kSums], db[kSums];
#pragma unroll
    for (int k = 0; k < kSums; ++k) dw[k] = db[k] = two(A(0), A(0));
    if constexpr (!kRegisters)
    {
#pragma unroll
        for (int k = 0; k < COLS; ++k) own[k * blockDim.x + threadIdx.x] = two(A(0), A(0));
    }
    const int64_t step = static_cast<int64_t>(gridDim.x) * groups;
    int64_t base = static_cast<int64_t>(blockIdx.x) * groups;
    Row next_x, next_g, weight;
    A next_mean = 0, next_rstd = 0;
    // pointers that walk along, where registers are left for them (4999 x 1001 in fp32: 19 us, 23 with products; 4096 x 16384 in bf16: 159 and 147)
    const T *x_from = static_cast<const T *>(a.x) + (base + mine) * a.x_stride, *g_from = static_cast<const T *>(a.dy) + (base + mine) * a.dy_stride;
    T *to = static_cast<T *>(a.y) + (base + mine) * a.y_stride;
    const int64_t x_step = step * a.x_stride, g_step = step * a.dy_stride, to_step = step * a.y_stride;
    const auto fetch = [&](int64_t row) {
        if (row >= a.rows) return;
        next_x.load(kRegisters ? x_from : static_cast<const T *>(a.x) + row * a.x_stride, lane, a.group, width);
        next_g.load(kRegisters ? g_from : static_cast<const T *>(a.dy) + row * a.dy_stride, lane, a.group, width);
        x_from += x_step;
        g_from += g_step;
        next_mean = static_cast<const A *>(a.mean)[row];
        next_rstd = static_cast<const A *>(a.rstd)[row];
    };
    fetch(base + mine);
    if (a.w != nullptr) weight.load(static_cast<const T *>(a.w), lane, a.group, width);
    else weight.fill(narrow2<T>(two(A(1), A(1))));
    for (; base < a.rows; base += step)
    {
        const int64_t row = base + mine;
        const bool there = row < a.rows;
        P x[COLS / 2], g[COLS / 2], sum_g = two(A(0), A(0)), sum_gx = sum_g;
        const A rstd = next_rstd;
        if (there)
        {
            const P means = two(next_mean, next_mean), scale = two(rstd, rstd);
#pragma unroll
            for (int k = 0; k < COLS / 2; ++k)
            {
                // columns behind the width have dy = 0 and weigh nothing
                const P dy = widen2<T>(next_g.pair[k]);
                x[k] = mul2(sub2(widen2<T>(next_x.pair[k]), means), scale);
                if constexpr (kRegisters)
                {
                    db[k] = add2(db[k], dy);
                    dw[k] = fma2(dy, x[k], dw[k]);
                }
                else
                {
                    P &w = own[k * blockDim.x + threadIdx.x], &b = own[(COLS / 2 + k) * blockDim.x + threadIdx.x];
                    w = fma2(dy, x[k], w);
                    b = add2(b, dy);
                }
                g[k] = mul2(dy, widen2<T>(weight.pair[k]));
                sum_g = add2(sum_g, g[k]);
                sum_gx = fma2(g[k], x[k], sum_gx);
            }
        }
        fetch(row + step);
        A s[2] = {first_of(sum_g) + second_of(sum_g), first_of(sum_gx) + second_of(sum_gx)};
        group_sum(s, slots[turn] + slot, a.group);
        turn ^= 1;
        if (there)
        {
            const P mean_g = two(s[0] * inv, s[0] * inv), mean_gx = two(-s[1] * inv, -s[1] * inv), scale = two(rstd, rstd);
            Row out;
#pragma unroll
            for (int k = 0; k < COLS / 2; ++k) out.pair[k] = narrow2<T>(mul2(scale, fma2(x[k], mean_gx, sub2(g[k], mean_g))));
            out.store(kRegisters ? to : static_cast<T *>(a.y) + row * a.y_stride, lane, a.group, width);
            to += to_step;
        }
    }
    if (a.partial == nullptr) return;
    A *out = static_cast<A *>(a.partial) + static_cast<int64_t>(blockIdx.x) * 2 * width;
    if constexpr (!kRegisters)
    {
        // rows this wide have one group: the columns are this thread's alone
#pragma unroll
        for (int k = 0; k < COLS / 2; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e)
            {
                const int c = Row::column(k, e, lane, a.group);
                if (c >= width) continue;
                const P w = own[k * blockDim.x + threadIdx.x], b = own[(COLS / 2 + k) * blockDim.x + threadIdx.x];
                out[c] = e ? second_of(w) : first_of(w);
                out[width + c] = e ? second_of(b) : first_of(b);
            }
        return;
    }
    else
    {
        // the groups' sums in ascending order
        A *to = groups == 1 ? out : sums + static_cast<size_t>(mine) * 2 * width;
#pragma unroll
        for (int k = 0; k < kSums; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e)
            {
                const int c = Row::column(k, e, lane, a.group);
                if (c >= width) continue;
                to[c] = e ? second_of(dw[k]) : first_of(dw[k]);
                to[width + c] = e ? second_of(db[k]) : first_of(db[k]);
            }
        if (groups == 1) return;
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * width; c += blockDim.x)
        {
            A s = sums[c];
#pragma unroll 4
            for (int one = 1; one < groups; ++one) s += sums[one * 2 * width + c];
            out[c] = s;
        }
    }
}

template <class T>
__global__ void __launch_bounds__(kWideThreads) norm_gradient_wide_kernel(NormArgs a)
{
    using A = typename Element<T>::Acc;
    __shared__ __align__(16) A slot[2 * kWideThreads / 32];
    const int64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride, *dy = static_cast<const T *>(a.dy) + row * a.dy_stride;
    const A inv = A(1) / static_cast<A>(a.width), mean = static_cast<const A *>(a.mean)[row], rstd = static_cast<const A *>(a.rstd)[row];
    A s[2] = {0, 0};
    for (int64_t c = threadIdx.x; c < a.width; c += kWideThreads)
    {
        const A g = widen(dy[c]) * (a.w != nullptr ? static_cast<A>(widen(static_cast<const T *>(a.w)[c])) : A(1));
        s[0] += g;
        s[1] += g * ((widen(x[c]) - mean) * rstd);
    }
    group_sum(s, slot, kWideThreads);
    s[0] *= inv;
    s[1] *= inv;
    T *dx = static_cast<T *>(a.y) + row * a.y_stride;
    for (int64_t c = threadIdx.x; c < a.width; c += kWideThreads)
    {
        const A g = widen(dy[c]) * (a.w != nullptr ? static_cast<A>(widen(static_cast<const T *>(a.w)[c])) : A(1));
        dx[c] = narrow<T>(rstd * (g - s[0] - (widen(x[c]) - mean) * rstd * s[1]));
    }
}

// The column sums of wide rows: CTA (column tile, slab of rows), a thread per column.
template <class T>
__global__ void __launch_bounds__(256) norm_columns_wide_kernel(NormArgs a)
{
    using A = typename Element<T>::Acc;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (c >= a.width) return;
    A dw = 0, db = 0;
    for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y)
    {
        const A g = widen(static_cast<const T *>(a.dy)[r * a.dy_stride + c]);
        db += g;
        dw += g * ((widen(static_cast<const T *>(a.x)[r * a.x_stride + c]) - static_cast<const A *>(a.mean)[r]) * static_cast<const A *>(a.rstd)[r]);
    }
    A *out = static_cast<A *>(a.partial) + static_cast<int64_t>(blockIdx.y) * 2 * a.width;
    out[c] = dw;
    out[a.width + c] = db;
}

// out[c] = sum over the parts, in ascending order within each of the 32 threads of a column and then over those threads.
template <class A>
__global__ void __launch_bounds__(1024) norm_combine_kernel(const A *partial, A *dw, A *db, int parts, int64_t width)
{
    __shared__ A sums[32][33];
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x;      // over 2 * width: the sums of dw, then those of db
    A s = 0;
    if (c < 2 * width)
#pragma unroll 8
        for (int p = threadIdx.y; p < parts; p += 32) s += partial[static_cast<int64_t>(p) * 2 * width + c];
    sums[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y != 0 || c >= 2 * width) return;
    for (int k = 1; k < 32; ++k) s += sums[k][threadIdx.x];
    if (c < width)
    {
        if (dw != nullptr) dw[c] = s;
    }
    else if (db != nullptr) db[c - width] = s;
}

// How rows of this width are cut up.
struct Shape
{
    int vec, cols, group, threads;      // cols = 0: the wide kernels
    int groups() const { return threads / group; }
};

int sms() { return sm_count() > 0 ? sm_count() : 148; }

// Columns a thread: as many as give it 64 bytes of a row (the gradient, which reads two rows: 32), at least 8, as long as the threads
// then still fill the GPU; fewer for few rows, down to 8; more when 512 threads would not cover the row.  (16384 x 4096 in bf16, 8 / 16 / 32
// columns: forward 119 / 64 / 52 us, gradient 117 / 93 us with 8 / 16; forward in fp32 130 / 91 us with 8 / 16.)
Shape norm_shape(int type, int64_t rows, int64_t width, bool vectors, bool gradient)
{
    Shape s;
    s.vec = vectors ? static_cast<int>(16 / element_bytes(type)) : 1;
    const int most = type == ACRO_B200_F64 ? 16 : 32;
    s.cols = std::max(8, static_cast<int>((gradient ? 32 : 64) / element_bytes(type)));
    while (s.cols > 8 && rows * width / s.cols < static_cast<int64_t>(sms()) * 512) s.cols /= 2;
    while (s.cols < most && width > static_cast<int64_t>(s.cols) * kMaxThreads) s.cols *= 2;
    if (width > static_cast<int64_t>(s.cols) * kMaxThreads)
    {
        s.cols = 0;
        s.group = s.threads = kWideThreads;
        return s;
    }
    const int lanes = static_cast<int>((width + s.cols - 1) / s.cols);
    s.group = 1;
    while (s.group < lanes && s.group < 32) s.group *= 2;
    if (lanes > 32) s.group = (lanes + 31) / 32 * 32;
    s.threads = s.group <= 128 ? 256 / s.group * s.group : s.group;
    return s;
}

// CTAs that walk over the rows: as many as are resident at once, and no more than rows need.
int norm_grid(int64_t rows, const Shape &s, int per_sm)
{
    const int64_t most = static_cast<int64_t>(sms()) * std::max(1, per_sm), need = (rows + s.groups() - 1) / s.groups();
    return static_cast<int>(std::max<int64_t>(1, std::min(most, need)));
}

// Rows of partial sums: the gradient's CTAs (512 threads an SM: 768 and 1024 were slower in every shape measured), or the slabs of rows
// of the wide rows' column sums.
int gradient_parts(int64_t rows, const Shape &s)
{
    if (s.cols == 0) return static_cast<int>(std::min<int64_t>(rows, sms()));
    return norm_grid(rows, s, 512 / s.threads);
}

template <class T, int VEC, int COLS, int THREADS>
int launch(const Shape &s, const NormArgs &a, bool gradient, cudaStream_t stream)
{
    const char *name = gradient ? "acro_b200_layer_norm_backward" : "acro_b200_layer_norm";
    if (!gradient)
    {
        int resident = 1;
        const cudaError_t status = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, norm_kernel<T, VEC, COLS, THREADS>, s.threads, 0);
        if (status != cudaSuccess) return fail_cuda(status, name);
        norm_kernel<T, VEC, COLS, THREADS><<<norm_grid(a.rows, s, resident), s.threads, 0, stream>>>(a);
        return launch_status(name);
    }
    // gradients of 32 columns a thread have CTAs of more than 256 threads
    if constexpr (COLS <= 16 || THREADS > 256)
    {
        const int smem = COLS > 16 ? COLS * s.threads * 2 * static_cast<int>(sizeof(typename Element<T>::Acc))
                                   : s.groups() > 1 ? s.groups() * 2 * static_cast<int>(a.width * sizeof(typename Element<T>::Acc)) : 0;
        cudaError_t status = allow_dynamic_smem(norm_gradient_kernel<T, VEC, COLS, THREADS>, smem);
        if (status != cudaSuccess) return fail_cuda(status, name);
        norm_gradient_kernel<T, VEC, COLS, THREADS><<<gradient_parts(a.rows, s), s.threads, smem, stream>>>(a);
    }
    return launch_status(name);
}

template <class T, int VEC>
int launch_norm(const Shape &s, const NormArgs &a, bool gradient, cudaStream_t stream)
{
    if (s.threads <= 256)
    {
        if (s.cols == 8) return launch<T, VEC, 8, 256>(s, a, gradient, stream);
        if (s.cols == 16) return launch<T, VEC, 16, 256>(s, a, gradient, stream);
        if constexpr (sizeof(T) == 2) return launch<T, VEC, 32, 256>(s, a, gradient, stream);
    }
    if (s.cols == 8) return launch<T, VEC, 8, 512>(s, a, gradient, stream);
    if (s.cols == 16) return launch<T, VEC, 16, 512>(s, a, gradient, stream);
    if constexpr (sizeof(T) < 8) return launch<T, VEC, 32, 512>(s, a, gradient, stream);
    return fail_unsupported("layer norm: no kernel for this shape");
}

template <class T>
int forward_of(const Shape &s, const NormArgs &a, cudaStream_t stream)
{
    if (s.cols == 0)
    {
        norm_wide_kernel<T><<<static_cast<unsigned>(a.rows), kWideThreads, 0, stream>>>(a);
        return launch_status("acro_b200_layer_norm");
    }
    return s.vec == 1 ? launch_norm<T, 1>(s, a, false, stream) : launch_norm<T, 16 / sizeof(T)>(s, a, false, stream);
}

template <class T>
int gradient_of(const Shape &s, const NormArgs &a, void *dw, void *db, cudaStream_t stream)
{
    using A = typename Element<T>::Acc;
    const int parts = gradient_parts(a.rows, s);
    if (s.cols == 0)
    {
        norm_gradient_wide_kernel<T><<<static_cast<unsigned>(a.rows), kWideThreads, 0, stream>>>(a);
        if (a.partial != nullptr)
            norm_columns_wide_kernel<T><<<dim3(static_cast<unsigned>((a.width + 255) / 256), parts), 256, 0, stream>>>(a);
    }
    else
    {
        const int status = s.vec == 1 ? launch_norm<T, 1>(s, a, true, stream) : launch_norm<T, 16 / sizeof(T)>(s, a, true, stream);
        if (status != ACRO_B200_OK) return status;
    }
    if (a.partial != nullptr)
        norm_combine_kernel<A><<<static_cast<unsigned>((2 * a.width + 31) / 32), dim3(32, 32), 0, stream>>>(
            static_cast<const A *>(a.partial), static_cast<A *>(dw), static_cast<A *>(db), parts, a.width);
    return launch_status("acro_b200_layer_norm_backward");
}

// Do packs of 16 bytes fit: rows that start on 16-byte boundaries and whose width is a multiple of the pack?
bool packs_fit(int type, int64_t width, std::initializer_list<const void *> pointers, std::initializer_list<int64_t> strides)
{
    const int64_t n = static_cast<int64_t>(16 / element_bytes(type));
    if (width % n != 0) return false;
    for (const void *p : pointers)
        if (!aligned16(p)) return false;
    for (int64_t s : strides)
        if (s % n != 0) return false;
    return true;
}

const char *shape_fault(int type, int64_t rows, int64_t width)
{
    if (!known_type(type)) return "unknown element type";
    if (rows < 0 || rows > INT32_MAX) return "the number of rows is not in 0 .. 2^31-1";
    if (width < 1 || width > (int64_t(1) << 30)) return "the width is not in 1 .. 2^30";
    return nullptr;
}

}

extern "C" {

int acro_b200_layer_norm(int type, const void *x, int64_t x_stride, const void *weight, const void *bias, void *y, int64_t y_stride, void *mean,
                         void *rstd, int64_t rows, int64_t width, double eps, void *stream)
{
    if (const char *fault = shape_fault(type, rows, width)) return fail_invalid(std::string("acro_b200_layer_norm: ") + fault);
    if (!(eps >= 0)) return fail_invalid("acro_b200_layer_norm: eps is negative or not a number");
    if (rows == 0) return ACRO_B200_OK;
    if (x == nullptr || y == nullptr) return fail_invalid("acro_b200_layer_norm: null pointer");
    if (x_stride < width || y_stride < width) return fail_invalid("acro_b200_layer_norm: rows overlap (a row stride is smaller than the width)");
    if (x == y && x_stride != y_stride) return fail_invalid("acro_b200_layer_norm: in place, but with different row strides");
    if (mean != nullptr && mean == rstd) return fail_invalid("acro_b200_layer_norm: mean and rstd take the same place");
    if (!aligned_to({x, weight, bias, y}, element_bytes(type)) || !aligned_to({mean, rstd}, statistic_bytes(type)))
        return fail_invalid("acro_b200_layer_norm: a pointer is not aligned to its elements");
    if (!all_on_device({x, weight, bias, y, mean, rstd})) return fail_invalid("acro_b200_layer_norm: a pointer is not memory of the current device");
    NormArgs a = {x, weight, bias, nullptr, y, mean, rstd, nullptr, rows, width, x_stride, y_stride, 0, eps, 0};
    const Shape s = norm_shape(type, rows, width, packs_fit(type, width, {x, weight, bias, y}, {x_stride, y_stride}), false);
    a.group = s.group;
    cudaStream_t st = as_stream(stream);
    if (type == ACRO_B200_F64) return forward_of<double>(s, a, st);
    if (type == ACRO_B200_F32) return forward_of<float>(s, a, st);
    return type == ACRO_B200_BF16 ? forward_of<__nv_bfloat16>(s, a, st) : forward_of<__half>(s, a, st);
}

size_t acro_b200_layer_norm_backward_scratch_bytes(int type, int64_t rows, int64_t width)
{
    if (shape_fault(type, rows, width) != nullptr || rows == 0) return 0;
    // independent of whether packs of 16 bytes will fit
    const Shape s = norm_shape(type, rows, width, true, true);
    return static_cast<size_t>(gradient_parts(rows, s)) * 2 * static_cast<size_t>(width) * statistic_bytes(type);
}

int acro_b200_layer_norm_backward(int type, const void *dy, int64_t dy_stride, const void *x, int64_t x_stride, const void *weight, const void *mean,
                                  const void *rstd, void *dx, int64_t dx_stride, void *dweight, void *dbias, int64_t rows, int64_t width, void *scratch,
                                  size_t scratch_bytes, void *stream)
{
    const char *name = "acro_b200_layer_norm_backward: ";
    if (const char *fault = shape_fault(type, rows, width)) return fail_invalid(std::string(name) + fault);
    cudaStream_t st = as_stream(stream);
    if (!aligned_to({dy, x, weight, dx}, element_bytes(type)) || !aligned_to({mean, rstd, dweight, dbias}, statistic_bytes(type)))
        return fail_invalid(std::string(name) + "a pointer is not aligned to its elements");
    if (dweight != nullptr && dweight == dbias) return fail_invalid(std::string(name) + "dweight and dbias take the same place");
    if (rows == 0)
    {
        // sums over no rows
        if (!all_on_device({dweight, dbias}))
            return fail_invalid(std::string(name) + "a pointer is not memory of the current device");
        const size_t bytes = static_cast<size_t>(width) * statistic_bytes(type);
        if (dweight != nullptr && cudaMemsetAsync(dweight, 0, bytes, st) != cudaSuccess) return fail_cuda(cudaGetLastError(), name);
        if (dbias != nullptr && cudaMemsetAsync(dbias, 0, bytes, st) != cudaSuccess) return fail_cuda(cudaGetLastError(), name);
        return ACRO_B200_OK;
    }
    if (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr || dx == nullptr) return fail_invalid(std::string(name) + "null pointer");
    if (x_stride < width || dy_stride < width || dx_stride < width)
        return fail_invalid(std::string(name) + "rows overlap (a row stride is smaller than the width)");
    if ((dx == x && dx_stride != x_stride) || (dx == dy && dx_stride != dy_stride))
        return fail_invalid(std::string(name) + "in place, but with different row strides");
    if (!all_on_device({dy, x, weight, mean, rstd, dx, dweight, dbias}))
        return fail_invalid(std::string(name) + "a pointer is not memory of the current device");
    const Shape s = norm_shape(type, rows, width, packs_fit(type, width, {x, weight, dy, dx}, {x_stride, dy_stride, dx_stride}), true);
    const bool sums = dweight != nullptr || dbias != nullptr;
    if (sums && s.cols == 0 && (dx == x || dx == dy))
        return fail_invalid(std::string(name) + "rows wider than 16384 (fp64: 8192) cannot be overwritten in place (their column sums are a second walk)");
    if (sums && (scratch == nullptr || scratch_bytes < acro_b200_layer_norm_backward_scratch_bytes(type, rows, width)))
        return fail_invalid(std::string(name) + "scratch is smaller than acro_b200_layer_norm_backward_scratch_bytes");
    if (sums && (!aligned16(scratch) || !on_current_device(scratch)))
        return fail_invalid(std::string(name) + "scratch is not 16-byte aligned memory of the current device");
    NormArgs a = {x, weight, nullptr, dy, dx, const_cast<void *>(mean), const_cast<void *>(rstd), sums ? scratch : nullptr, rows, width, x_stride,
                  dx_stride, dy_stride, 0, s.group};
    if (type == ACRO_B200_F64) return gradient_of<double>(s, a, dweight, dbias, st);
    if (type == ACRO_B200_F32) return gradient_of<float>(s, a, dweight, dbias, st);
    return type == ACRO_B200_BF16 ? gradient_of<__nv_bfloat16>(s, a, dweight, dbias, st) : gradient_of<__half>(s, a, dweight, dbias, st);
}

}
