// Element types of the sequence operators (linear attention, layer norm): what is stored in 16, 32 or 64 bits and computed in 32 or 64.
#ifndef ACRO_B200_KERNELS_ELEMENT_CUH
#define ACRO_B200_KERNELS_ELEMENT_CUH

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <initializer_list>

#include "common.cuh"

namespace acro_b200_detail
{

// Acc: the type of sums, states and statistics.
template <class T> struct Element { using Acc = float; };
template <> struct Element<double> { using Acc = double; };

template <class T> __device__ __forceinline__ typename Element<T>::Acc widen(T x) { return x; }
template <> __device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float widen<__half>(__half x) { return __half2float(x); }

template <class T> __device__ __forceinline__ T narrow(typename Element<T>::Acc x) { return static_cast<T>(x); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half narrow<__half>(float x) { return __float2half_rn(x); }

// N elements that travel as one access of N * sizeof(T) bytes.
template <class T, int N> struct alignas(sizeof(T) * N) Pack { T x[N]; };

template <int BYTES> struct Word;
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<16> { using type = uint4; };

// The access itself (copying the struct moves its 16-bit elements one by one).
template <class T, int N> __device__ __forceinline__ Pack<T, N> load_pack(const T *from)
{
    using W = typename Word<sizeof(T) * N>::type;
    Pack<T, N> p;
    *reinterpret_cast<W *>(&p) = *reinterpret_cast<const W *>(from);
    return p;
}
template <class T, int N> __device__ __forceinline__ void store_pack(T *to, const Pack<T, N> &p)
{
    using W = typename Word<sizeof(T) * N>::type;
    *reinterpret_cast<W *>(to) = *reinterpret_cast<const W *>(&p);
}

// Two neighbouring values of a type of sums.  For fp32 they share a 64-bit register, and one instruction works on both.
typedef unsigned long long Two;
struct TwoWide { double first, second; };
template <class A> struct PairOf { using type = Two; };
template <> struct PairOf<double> { using type = TwoWide; };

__device__ __forceinline__ Two two(float x, float y)
{
    Two d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
    return d;
}
__device__ __forceinline__ Two two(uint32_t x, uint32_t y) { return two(__uint_as_float(x), __uint_as_float(y)); }
__device__ __forceinline__ TwoWide two(double x, double y) { return {x, y}; }
__device__ __forceinline__ float first_of(Two x) { return __uint_as_float(static_cast<uint32_t>(x)); }
__device__ __forceinline__ float second_of(Two x) { return __uint_as_float(static_cast<uint32_t>(x >> 32)); }
__device__ __forceinline__ double first_of(TwoWide x) { return x.first; }
__device__ __forceinline__ double second_of(TwoWide x) { return x.second; }
__device__ __forceinline__ Two fma2(Two a, Two b, Two c)
{
    Two d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ Two mul2(Two a, Two b)
{
    Two d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Two add2(Two a, Two b)
{
    Two d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Two sub2(Two a, Two b)
{
    Two d;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ TwoWide fma2(TwoWide a, TwoWide b, TwoWide c) { return {fma(a.first, b.first, c.first), fma(a.second, b.second, c.second)}; }
__device__ __forceinline__ TwoWide mul2(TwoWide a, TwoWide b) { return {a.first * b.first, a.second * b.second}; }
__device__ __forceinline__ TwoWide add2(TwoWide a, TwoWide b) { return {a.first + b.first, a.second + b.second}; }
__device__ __forceinline__ TwoWide sub2(TwoWide a, TwoWide b) { return {a.first - b.first, a.second - b.second}; }

__device__ __forceinline__ uint32_t pack_bf16(Two x)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(second_of(x)), "f"(first_of(x)));
    return r;
}
// The same, but finite values above the largest bf16 (and infinities) become that one: what is left of a finite value is finite.
__device__ __forceinline__ uint32_t pack_bf16_finite(Two x)
{
    uint32_t r;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(second_of(x)), "f"(first_of(x)));
    return r;
}
__device__ __forceinline__ Two unpack_bf16(uint32_t x) { return two(x << 16, x & 0xffff0000u); }

// Two neighbouring elements as they lie in memory.
template <class T> struct Raw { using type = uint32_t; };
template <> struct Raw<float> { using type = uint2; };
template <> struct Raw<double> { using type = double2; };

template <class T> __device__ __forceinline__ Two widen2(uint32_t x);
template <> __device__ __forceinline__ Two widen2<__nv_bfloat16>(uint32_t x) { return unpack_bf16(x); }
template <> __device__ __forceinline__ Two widen2<__half>(uint32_t x)
{
    Two d;
    asm("{\n"
        ".reg .b16 l, h;\n"
        ".reg .f32 x, y;\n"
        "mov.b32 {l, h}, %1;\n"
        "cvt.f32.f16 x, l;\n"
        "cvt.f32.f16 y, h;\n"
        "mov.b64 %0, {x, y};\n"
        "}\n"
        : "=l"(d)
        : "r"(x));
    return d;
}
template <class T> __device__ __forceinline__ Two widen2(uint2 x) { return two(x.x, x.y); }
template <class T> __device__ __forceinline__ TwoWide widen2(double2 x) { return {x.x, x.y}; }

template <class T> __device__ __forceinline__ typename Raw<T>::type narrow2(typename PairOf<typename Element<T>::Acc>::type x);
template <> __device__ __forceinline__ uint32_t narrow2<__nv_bfloat16>(Two x) { return pack_bf16(x); }
template <> __device__ __forceinline__ uint32_t narrow2<__half>(Two x)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(second_of(x)), "f"(first_of(x)));
    return r;
}
template <> __device__ __forceinline__ uint2 narrow2<float>(Two x) { return make_uint2(__float_as_uint(first_of(x)), __float_as_uint(second_of(x))); }
template <> __device__ __forceinline__ double2 narrow2<double>(TwoWide x) { return make_double2(x.first, x.second); }

// COLS columns of a row, as they lie in memory: those of thread `lane` of a group of `group` threads are the packs lane, lane + group, ...
// of VEC columns (VEC = 1: single elements, pair k from the elements 2 k and 2 k + 1 of this thread).  Columns from `width` on are zeros.
template <class T, int VEC, int COLS> struct RowPart
{
    static constexpr int kPairs = COLS / 2;
    typename Raw<T>::type pair[kPairs];

    static __device__ __forceinline__ int column(int k, int e, int lane, int group)
    {
        return VEC == 1 ? (2 * k + e) * group + lane : (k / (VEC > 1 ? VEC / 2 : 1) * group + lane) * VEC + k % (VEC > 1 ? VEC / 2 : 1) * 2 + e;
    }
    __device__ __forceinline__ void load(const T *row, int lane, int group, int width)
    {
        if constexpr (VEC == 1)
        {
#pragma unroll
            for (int k = 0; k < kPairs; ++k)
            {
                Pack<T, 2> p;
#pragma unroll
                for (int e = 0; e < 2; ++e)
                {
                    const int c = column(k, e, lane, group);
                    if (c < width) store_pack<T, 1>(&p.x[e], load_pack<T, 1>(row + c));
                    else p.x[e] = T(0.0f);
                }
                pair[k] = *reinterpret_cast<const typename Raw<T>::type *>(&p);
            }
        }
        else
        {
            using W = typename Word<sizeof(T) * VEC>::type;
#pragma unroll
            for (int q = 0; q < COLS / VEC; ++q)
            {
                const int c = (q * group + lane) * VEC;
                W w = {};
                if (c < width) w = *reinterpret_cast<const W *>(row + c);
#pragma unroll
                for (int i = 0; i < VEC / 2; ++i) pair[q * (VEC / 2) + i] = reinterpret_cast<const typename Raw<T>::type *>(&w)[i];
            }
        }
    }
    __device__ __forceinline__ void store(T *row, int lane, int group, int width) const
    {
        if constexpr (VEC == 1)
        {
#pragma unroll
            for (int k = 0; k < kPairs; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                {
                    const int c = column(k, e, lane, group);
                    if (c < width) store_pack<T, 1>(row + c, reinterpret_cast<const Pack<T, 1> *>(&pair[k])[e]);
                }
        }
        else
        {
            using W = typename Word<sizeof(T) * VEC>::type;
#pragma unroll
            for (int q = 0; q < COLS / VEC; ++q)
            {
                const int c = (q * group + lane) * VEC;
                if (c >= width) continue;
                W w;
#pragma unroll
                for (int i = 0; i < VEC / 2; ++i) reinterpret_cast<typename Raw<T>::type *>(&w)[i] = pair[q * (VEC / 2) + i];
                *reinterpret_cast<W *>(row + c) = w;
            }
        }
    }
    __device__ __forceinline__ void fill(typename Raw<T>::type value)
    {
#pragma unroll
        for (int k = 0; k < kPairs; ++k) pair[k] = value;
    }
};

inline size_t element_bytes(int type) { return type == ACRO_B200_F64 ? 8 : type == ACRO_B200_F32 ? 4 : 2; }
inline size_t statistic_bytes(int type) { return type == ACRO_B200_F64 ? 8 : 4; }
inline bool known_type(int type) { return type >= ACRO_B200_F64 && type <= ACRO_B200_F16; }

// Is `p` memory that kernels on the current device can be given?  Memory of another device is refused: a kernel of this
// device would read it over the link or fault.  (Host memory that is mapped or managed passes.)
inline bool on_current_device(const void *p)
{
    cudaPointerAttributes a;
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaPointerGetAttributes(&a, p) != cudaSuccess)
    {
        cudaGetLastError();
        return false;
    }
    if (a.type == cudaMemoryTypeDevice) return a.device == dev;
    return a.type == cudaMemoryTypeManaged || (a.type == cudaMemoryTypeHost && a.devicePointer != nullptr);
}

// The same for several pointers, null ones aside.
inline bool all_on_device(std::initializer_list<const void *> pointers)
{
    for (const void *p : pointers)
        if (p != nullptr && !on_current_device(p)) return false;
    return true;
}

// Do these arrays start on a boundary of their elements?
inline bool aligned_to(std::initializer_list<const void *> pointers, size_t bytes)
{
    for (const void *p : pointers)
        if (reinterpret_cast<uintptr_t>(p) % bytes != 0) return false;
    return true;
}

}

#endif
