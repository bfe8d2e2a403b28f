// Layer norm of rows and its gradient.
//
//   mean = sum_f x_f / W,  rstd = 1 / sqrt(sum_f (x_f - mean)^2 / W + eps),  xhat = (x - mean) rstd,  y = xhat w + b
//   g = dy w,  dx = rstd (g - sum(g)/W - xhat sum(g xhat)/W),  dw_f = sum_rows dy xhat,  db_f = sum_rows dy
//
// Both are bound by HBM: 2 and 3 elements moved per entry against about ten operations.  So a row is read once, stays in
// registers between its moments and its result, and leaves once.  A row belongs to a group of G threads (whole warps); a CTA
// holds 256/G groups when rows are short.  The variance is the mean square of the centred entries (a second walk over the
// registers), not a difference of moments, which cancels for rows far from zero.
//
// The gradient's column sums run over all rows: a thread owns the same columns of every row that its group takes (rows r,
// r + groups, ...), so the sums over those rows stay in its registers; a group leaves one row of partial sums, and a second
// kernel adds the groups' rows in ascending order.  No atomics: the same bits on every run on one device.
#include "element.cuh"

#include <algorithm>

using namespace acro_b200_detail;

namespace
{

constexpr int kMaxThreads = 512;       // of one group; 32 columns a thread and two sums a column fit the registers of 512 threads
constexpr int kColumnsMax = 32;        // columns of one thread
constexpr int kWideThreads = 512;

struct NormArgs
{
    const void *x, *w, *b, *dy;
    void *y;                            // the result, or dx
    void *mean, *rstd;                  // written by the forward pass (or null), read by the gradient
    void *partial;                      // gradient: [groups][2][width] sums
    int64_t rows, width, x_stride, y_stride, dy_stride;
    double eps;
    int group;                          // threads of one row
};

// Sum over the threads of a row's group; `slot` is the group's own part of shared memory (one entry per warp), written and
// read between two barriers of the whole CTA.  Every thread of the CTA calls it.
template <int N, class A>
__device__ __forceinline__ void group_sum(A (&v)[N], A *slot, int group)
{
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    const int warps = group / 32;
    if (warps == 1) return;
    const int warp = (threadIdx.x % group) / 32;
    __syncthreads();                    // the previous sum's entries have been read
    if (threadIdx.x % 32 == 0)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) slot[warp * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0;
    for (int k = 0; k < warps; ++k)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += slot[k * N + i];
    }
}

// The columns of thread `lane` of a group of `group` threads: packs lane, lane + group, ... of VEC columns.
template <class T, int VEC, int COLS, class A>
__device__ __forceinline__ void load_row(A (&v)[COLS], const T *row, int lane, int group, int64_t width, A missing)
{
    Pack<T, VEC> p[COLS / VEC];
#pragma unroll
    for (int k = 0; k < COLS / VEC; ++k)
    {
        const int64_t c = (static_cast<int64_t>(k) * group + lane) * VEC;
        if (c < width) p[k] = *reinterpret_cast<const Pack<T, VEC> *>(row + c);
    }
#pragma unroll
    for (int k = 0; k < COLS / VEC; ++k)
    {
        const bool there = (static_cast<int64_t>(k) * group + lane) * VEC < width;
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[k * VEC + j] = there ? static_cast<A>(widen(p[k].x[j])) : missing;
    }
}

template <class T, int VEC, int COLS, class A>
__device__ __forceinline__ void store_row(const A (&v)[COLS], T *row, int lane, int group, int64_t width)
{
#pragma unroll
    for (int k = 0; k < COLS / VEC; ++k)
    {
        const int64_t c = (static_cast<int64_t>(k) * group + lane) * VEC;
        if (c >= width) continue;
        Pack<T, VEC> p;
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.x[j] = narrow<T>(v[k * VEC + j]);
        *reinterpret_cast<Pack<T, VEC> *>(row + c) = p;
    }
}

template <class T, int VEC, int COLS>
__global__ void __launch_bounds__(kMaxThreads) norm_kernel(NormArgs a)
{
    using A = typename Element<T>::Acc;
    __shared__ A slots[kMaxThreads / 32];
    const int groups = blockDim.x / a.group, mine = threadIdx.x / a.group, lane = threadIdx.x % a.group;
    A *slot = slots + mine * (a.group / 32);
    const int64_t row = static_cast<int64_t>(blockIdx.x) * groups + mine;
    const bool there = row < a.rows;
    const A inv = A(1) / static_cast<A>(a.width);
    A x[COLS];
    if (there) load_row<T, VEC, COLS>(x, static_cast<const T *>(a.x) + row * a.x_stride, lane, a.group, a.width, A(0));
    else
#pragma unroll
        for (int i = 0; i < COLS; ++i) x[i] = 0;
    A s[1] = {0};
#pragma unroll
    for (int i = 0; i < COLS; ++i) s[0] += x[i];
    group_sum(s, slot, a.group);
    const A mean = s[0] * inv;
    s[0] = 0;
#pragma unroll
    for (int k = 0; k < COLS / VEC; ++k)
    {
        if ((static_cast<int64_t>(k) * a.group + lane) * VEC >= a.width) continue;
#pragma unroll
        for (int j = 0; j < VEC; ++j)
        {
            x[k * VEC + j] -= mean;
            s[0] += x[k * VEC + j] * x[k * VEC + j];
        }
    }
    group_sum(s, slot, a.group);
    const A rstd = A(1) / sqrt(s[0] * inv + static_cast<A>(a.eps));
    if (!there) return;
    if (lane == 0)
    {
        if (a.mean != nullptr) static_cast<A *>(a.mean)[row] = mean;
        if (a.rstd != nullptr) static_cast<A *>(a.rstd)[row] = rstd;
    }
#pragma unroll
    for (int k = 0; k < COLS / VEC; ++k)
    {
        const int64_t c = (static_cast<int64_t>(k) * a.group + lane) * VEC;
        if (c >= a.width) continue;
        Pack<T, VEC> w, b;
        if (a.w != nullptr) w = *reinterpret_cast<const Pack<T, VEC> *>(static_cast<const T *>(a.w) + c);
        if (a.b != nullptr) b = *reinterpret_cast<const Pack<T, VEC> *>(static_cast<const T *>(a.b) + c);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
        {
            A v = x[k * VEC + j] * rstd;
            if (a.w != nullptr) v *= widen(w.x[j]);
            if (a.b != nullptr) v += widen(b.x[j]);
            x[k * VEC + j] = v;
        }
    }
    store_row<T, VEC, COLS>(x, static_cast<T *>(a.y) + row * a.y_stride, lane, a.group, a.width);
}

// Rows wider than a group's registers hold: three walks over the row, the later two mostly from L2.
template <class T>
__global__ void __launch_bounds__(kWideThreads) norm_wide_kernel(NormArgs a)
{
    using A = typename Element<T>::Acc;
    __shared__ A slot[kWideThreads / 32];
    const int64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const A inv = A(1) / static_cast<A>(a.width);
    A s[1] = {0};
    for (int64_t c = threadIdx.x; c < a.width; c += kWideThreads) s[0] += widen(x[c]);
    group_sum(s, slot, kWideThreads);
    const A mean = s[0] * inv;
    s[0] = 0;
    for (int64_t c = threadIdx.x; c < a.width; c += kWideThreads)
    {
        const A d = widen(x[c]) - mean;
        s[0] += d * d;
    }
    group_sum(s, slot, kWideThreads);
    const A rstd = A(1) / sqrt(s[0] * inv + static_cast<A>(a.eps));
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

template <class T, int VEC, int COLS>
__global__ void __launch_bounds__(kMaxThreads) norm_gradient_kernel(NormArgs a)
{
    using A = typename Element<T>::Acc;
    __shared__ A slots[2 * kMaxThreads / 32];
    const int groups = blockDim.x / a.group, mine = threadIdx.x / a.group, lane = threadIdx.x % a.group;
    A *slot = slots + mine * (a.group / 32) * 2;
    const A inv = A(1) / static_cast<A>(a.width);
    A dw[COLS], db[COLS];
#pragma unroll
    for (int i = 0; i < COLS; ++i) dw[i] = db[i] = 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * groups;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * groups; base < a.rows; base += step)
    {
        const int64_t row = base + mine;
        const bool there = row < a.rows;
        A x[COLS], g[COLS], s[2] = {0, 0}, rstd = 0;
        if (there)
        {
            load_row<T, VEC, COLS>(x, static_cast<const T *>(a.x) + row * a.x_stride, lane, a.group, a.width, A(0));
            load_row<T, VEC, COLS>(g, static_cast<const T *>(a.dy) + row * a.dy_stride, lane, a.group, a.width, A(0));
            const A mean = static_cast<const A *>(a.mean)[row];
            rstd = static_cast<const A *>(a.rstd)[row];
#pragma unroll
            for (int k = 0; k < COLS / VEC; ++k)
            {
                const int64_t c = (static_cast<int64_t>(k) * a.group + lane) * VEC;
                if (c >= a.width) continue;
                Pack<T, VEC> w;
                if (a.w != nullptr) w = *reinterpret_cast<const Pack<T, VEC> *>(static_cast<const T *>(a.w) + c);
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                {
                    const int i = k * VEC + j;
                    x[i] = (x[i] - mean) * rstd;
                    db[i] += g[i];
                    dw[i] += g[i] * x[i];
                    if (a.w != nullptr) g[i] *= widen(w.x[j]);
                    s[0] += g[i];
                    s[1] += g[i] * x[i];
                }
            }
        }
        group_sum(s, slot, a.group);
        if (there)
        {
            s[0] *= inv;
            s[1] *= inv;
#pragma unroll
            for (int i = 0; i < COLS; ++i) x[i] = rstd * (g[i] - s[0] - x[i] * s[1]);
            store_row<T, VEC, COLS>(x, static_cast<T *>(a.y) + row * a.y_stride, lane, a.group, a.width);
        }
    }
    if (a.partial == nullptr) return;
    A *out = static_cast<A *>(a.partial) + (static_cast<int64_t>(blockIdx.x) * groups + mine) * 2 * a.width;
#pragma unroll
    for (int k = 0; k < COLS / VEC; ++k)
    {
        const int64_t c = (static_cast<int64_t>(k) * a.group + lane) * VEC;
        if (c >= a.width) continue;
#pragma unroll
        for (int j = 0; j < VEC; ++j)
        {
            out[c + j] = dw[k * VEC + j];
            out[a.width + c + j] = db[k * VEC + j];
        }
    }
}

template <class T>
__global__ void __launch_bounds__(kWideThreads) norm_gradient_wide_kernel(NormArgs a)
{
    using A = typename Element<T>::Acc;
    __shared__ A slot[2 * kWideThreads / 32];
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

// out[c] = sum over the parts, in ascending order within each of the 16 threads of a column and then over those threads.
template <class A>
__global__ void __launch_bounds__(512) norm_combine_kernel(const A *partial, A *dw, A *db, int parts, int64_t width)
{
    __shared__ A sums[16][33];
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x;      // over 2 * width: the sums of dw, then those of db
    A s = 0;
    if (c < 2 * width)
        for (int p = threadIdx.y; p < parts; p += 16) s += partial[static_cast<int64_t>(p) * 2 * width + c];
    sums[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y != 0 || c >= 2 * width) return;
    for (int k = 1; k < 16; ++k) s += sums[k][threadIdx.x];
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

// Columns a thread: 8, 16 or 32 of them, by whether a group of at most 512 threads then covers the row.
Shape norm_shape(int type, int64_t width, bool vectors)
{
    Shape s;
    s.vec = vectors ? static_cast<int>(16 / element_bytes(type)) : 1;
    s.cols = width <= 8 * kMaxThreads ? 8 : width <= 16 * kMaxThreads ? 16 : 32;
    if (width > static_cast<int64_t>(kColumnsMax) * kMaxThreads) s.cols = 0;
    if (s.cols == 0)
    {
        s.group = s.threads = kWideThreads;
        return s;
    }
    s.group = static_cast<int>((width + s.cols - 1) / s.cols + 31) / 32 * 32;
    s.threads = s.group <= 128 ? 256 / s.group * s.group : s.group;
    return s;
}

// CTAs of the gradient (and of the wide rows' column sums): enough to fill the GPU, few enough that their partial sums stay
// small against the rows.
int gradient_parts(int64_t rows, const Shape &s)
{
    const int sms = sm_count() > 0 ? sm_count() : 148;
    const int64_t most = static_cast<int64_t>(sms) * (s.cols == 0 ? 1 : std::max(1, 1024 / s.threads));
    const int64_t need = s.cols == 0 ? rows : (rows + s.groups() - 1) / s.groups();
    return static_cast<int>(std::max<int64_t>(1, std::min(most, need)));
}

template <class T, int VEC>
void launch_norm(const Shape &s, const NormArgs &a, bool gradient, int grid, cudaStream_t stream)
{
    if (gradient)
    {
        if (s.cols == 8) norm_gradient_kernel<T, VEC, 8><<<grid, s.threads, 0, stream>>>(a);
        else if (s.cols == 16) norm_gradient_kernel<T, VEC, 16><<<grid, s.threads, 0, stream>>>(a);
        else norm_gradient_kernel<T, VEC, 32><<<grid, s.threads, 0, stream>>>(a);
    }
    else
    {
        if (s.cols == 8) norm_kernel<T, VEC, 8><<<grid, s.threads, 0, stream>>>(a);
        else if (s.cols == 16) norm_kernel<T, VEC, 16><<<grid, s.threads, 0, stream>>>(a);
        else norm_kernel<T, VEC, 32><<<grid, s.threads, 0, stream>>>(a);
    }
}

template <class T>
int forward_of(const Shape &s, const NormArgs &a, cudaStream_t stream)
{
    const int64_t grid = s.cols == 0 ? a.rows : (a.rows + s.groups() - 1) / s.groups();
    if (s.cols == 0) norm_wide_kernel<T><<<static_cast<unsigned>(grid), kWideThreads, 0, stream>>>(a);
    else if (s.vec == 1) launch_norm<T, 1>(s, a, false, static_cast<int>(grid), stream);
    else launch_norm<T, 16 / sizeof(T)>(s, a, false, static_cast<int>(grid), stream);
    return launch_status("acro_b200_layer_norm");
}

template <class T>
int gradient_of(const Shape &s, const NormArgs &a, void *dw, void *db, cudaStream_t stream)
{
    using A = typename Element<T>::Acc;
    const int parts = gradient_parts(a.rows, s);
    int rows_of_sums = parts * s.groups();
    if (s.cols == 0)
    {
        norm_gradient_wide_kernel<T><<<static_cast<unsigned>(a.rows), kWideThreads, 0, stream>>>(a);
        if (a.partial != nullptr)
            norm_columns_wide_kernel<T><<<dim3(static_cast<unsigned>((a.width + 255) / 256), parts), 256, 0, stream>>>(a);
        rows_of_sums = parts;
    }
    else if (s.vec == 1) launch_norm<T, 1>(s, a, true, parts, stream);
    else launch_norm<T, 16 / sizeof(T)>(s, a, true, parts, stream);
    if (a.partial != nullptr)
        norm_combine_kernel<A><<<static_cast<unsigned>((2 * a.width + 31) / 32), dim3(32, 16), 0, stream>>>(
            static_cast<const A *>(a.partial), static_cast<A *>(dw), static_cast<A *>(db), rows_of_sums, a.width);
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
    if (!on_current_device(x) || !on_current_device(y)) return fail_invalid("acro_b200_layer_norm: a pointer is not memory of the current device");
    NormArgs a = {x, weight, bias, nullptr, y, mean, rstd, nullptr, rows, width, x_stride, y_stride, 0, eps, 0};
    const Shape s = norm_shape(type, width, packs_fit(type, width, {x, weight, bias, y}, {x_stride, y_stride}));
    a.group = s.group;
    cudaStream_t st = as_stream(stream);
    if (type == ACRO_B200_F64) return forward_of<double>(s, a, st);
    if (type == ACRO_B200_F32) return forward_of<float>(s, a, st);
    return type == ACRO_B200_BF16 ? forward_of<__nv_bfloat16>(s, a, st) : forward_of<__half>(s, a, st);
}

size_t acro_b200_layer_norm_backward_scratch_bytes(int type, int64_t rows, int64_t width)
{
    if (shape_fault(type, rows, width) != nullptr || rows == 0) return 0;
    size_t most = 0;
    for (int vectors = 0; vectors < 2; ++vectors)
    {
        const Shape s = norm_shape(type, width, vectors != 0);
        const size_t sums = static_cast<size_t>(gradient_parts(rows, s)) * (s.cols == 0 ? 1 : s.groups());
        most = std::max(most, sums * 2 * static_cast<size_t>(width) * statistic_bytes(type));
    }
    return most;
}

int acro_b200_layer_norm_backward(int type, const void *dy, int64_t dy_stride, const void *x, int64_t x_stride, const void *weight, const void *mean,
                                  const void *rstd, void *dx, int64_t dx_stride, void *dweight, void *dbias, int64_t rows, int64_t width, void *scratch,
                                  size_t scratch_bytes, void *stream)
{
    const char *name = "acro_b200_layer_norm_backward: ";
    if (const char *fault = shape_fault(type, rows, width)) return fail_invalid(std::string(name) + fault);
    cudaStream_t st = as_stream(stream);
    if (rows == 0)
    {
        // sums over no rows
        if ((dweight != nullptr && !on_current_device(dweight)) || (dbias != nullptr && !on_current_device(dbias)))
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
    if (!on_current_device(dy) || !on_current_device(x) || !on_current_device(dx))
        return fail_invalid(std::string(name) + "a pointer is not memory of the current device");
    const Shape s = norm_shape(type, width, packs_fit(type, width, {x, weight, dy, dx}, {x_stride, dy_stride, dx_stride}));
    const bool sums = dweight != nullptr || dbias != nullptr;
    if (sums && s.cols == 0 && (dx == x || dx == dy))
        return fail_invalid(std::string(name) + "rows wider than 16384 cannot be overwritten in place (their column sums are a second walk)");
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
