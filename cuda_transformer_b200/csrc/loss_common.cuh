// loss_common.cuh: what the losses share: the workspace, the element types, block reductions
// and the argument checks of a matrix.
#pragma once

#include <cuda_bf16.h>

#include <climits>
#include <cmath>

#include "internal.cuh"

namespace b200amp
{

// Zeroed once by the caller; every kernel leaves the counters at zero again, so graph replays
// need no memset. The losses have fields of their own, so one workspace serves a whole step.
struct LossWorkspace
{
    unsigned int distill_ticket;    // blocks finished so far; the last one resets it
    unsigned int balance_ticket;
    unsigned int rows_counted;      // balance: rows that count
    unsigned int beyond;            // balance: some choice named an expert beyond the last
    unsigned int pad[12];
    unsigned int counts[B200AMP_MAX_EXPERTS];
    double partial[2368];           // balance: one sum per block
};
static_assert(sizeof(LossWorkspace) <= B200AMP_LOSS_WORKSPACE_BYTES, "the workspace has a published size");

inline int dtype_size(int dtype)
{
    return dtype == B200AMP_F32 ? 4 : 2;
}

inline bool dtype_known(int dtype)
{
    return dtype == B200AMP_F16 || dtype == B200AMP_BF16 || dtype == B200AMP_F32;
}

#ifdef __CUDACC__

__device__ __forceinline__ float to_float(__half v)
{
    return __half2float(v);
}
__device__ __forceinline__ float to_float(__nv_bfloat16 v)
{
    return __bfloat162float(v);
}
__device__ __forceinline__ float to_float(float v)
{
    return v;
}

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v)
{
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v)
{
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ float from_float<float>(float v)
{
    return v;
}

// element i of an array of a type known at run time only (a record of k values a row)
__device__ __forceinline__ float load_typed(const void *p, int dtype, long long i)
{
    if (dtype == B200AMP_F32)
    {
        return static_cast<const float *>(p)[i];
    }
    if (dtype == B200AMP_F16)
    {
        return __half2float(static_cast<const __half *>(p)[i]);
    }
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}

// 2^x by the special function unit (2 ulp; results below 2^-126 become 0)
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// NaN wins, unlike fmaxf: a row that holds one has no maximum
__device__ __forceinline__ float max_nan(float a, float b)
{
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

__device__ __forceinline__ float warp_max_nan(float v)
{
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1)
    {
        v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, offset));
    }
    return v;
}

// Sums over the block, the warps' shares added in warp order by every thread. scratch: shared memory
// for one value a warp, free again when the call returns. Every thread of the block must call these.
template <int THREADS>
__device__ __forceinline__ double block_sum_f64(double v, double *scratch)
{
    v = warp_sum_f64(v);
    if ((threadIdx.x & 31) == 0)
    {
        scratch[threadIdx.x >> 5] = v;
    }
    __syncthreads();
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++)
    {
        total += scratch[w];
    }
    __syncthreads();
    return total;
}

// True (in every thread) for the block that takes the last ticket of `blocks`: all that the other
// blocks wrote before theirs is visible to it. The ticket is reset for the next launch.
__device__ __forceinline__ bool take_last_ticket(unsigned int *ticket, unsigned int blocks, int *shared_flag)
{
    __syncthreads();
    if (threadIdx.x == 0)
    {
        __threadfence();                        // this block's results before the ticket
        const unsigned int t = atomicAdd(ticket, 1u);
        *shared_flag = (t == blocks - 1) ? 1 : 0;
        if (t == blocks - 1)
        {
            *ticket = 0;
        }
    }
    __syncthreads();
    if (!*shared_flag)
    {
        return false;
    }
    __threadfence();                            // the other blocks' results after the ticket
    return true;
}

#endif // __CUDACC__

} // namespace b200amp
