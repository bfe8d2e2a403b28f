// Element types of the sequence operators (linear attention, layer norm): what is stored in 16, 32 or 64 bits and computed in 32 or 64.
#ifndef ACRO_B200_KERNELS_ELEMENT_CUH
#define ACRO_B200_KERNELS_ELEMENT_CUH

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

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

}

#endif
