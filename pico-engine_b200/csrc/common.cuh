// Shared helpers of the sm_100a kernels: element types, loads that convert to float,
// reductions, and the calling convention of the exported launchers.
//
// Every exported function is `extern "C" int pe_<name>(..., void* stream)`: it takes raw
// device pointers and sizes, launches on the given CUDA stream and returns 0 or a
// cudaError_t value (sizes a kernel does not take are refused with PE_ERR_UNSUPPORTED
// before anything is launched).  dtype codes: 0 = float32, 1 = bfloat16.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#define PE_F32 0
#define PE_BF16 1
#define PE_ERR_UNSUPPORTED 10001   // sizes or dtypes this kernel does not take
#define PE_PAGE 64                 // tokens in one page of the key/value cache

typedef __nv_bfloat16 bf16;

#define PE_LAUNCH_CHECK() do { cudaError_t e_ = cudaGetLastError(); if (e_ != cudaSuccess) return (int)e_; } while (0)
#define PE_TRY(call) do { cudaError_t e_ = (call); if (e_ != cudaSuccess) return (int)e_; } while (0)

// Programmatic dependent launch.  Every kernel of this library is launched so that it may start
// while its predecessor in the stream is still running (its blocks fill SMs the predecessor no
// longer needs), and every kernel calls pdl_wait() before it touches anything an earlier kernel
// wrote and before it writes anything: the wait returns when the predecessor has finished and
// its writes are visible.  What a kernel does before the wait (reading weights, which no
// kernel writes) overlaps the predecessor's tail.  pdl_launch_dependents() at a kernel's start
// lets its own successor be scheduled as early as possible.  Because a kernel can be resident
// while its predecessor still writes, kernel parameters are not declared __restrict__ (which
// would let the compiler read them through the non-coherent path).
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// The thread of a warp that issues for it (products on the tensor cores and their commits); the whole warp calls.
__device__ __forceinline__ unsigned pe_elect() {
    unsigned r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
    return r;
}
// SMs of the device, for grids whose blocks stay.
inline int pe_sm_count() {
    static int n = 0;
    if (!n) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    }
    return n;
}

// Lets a kernel's launches ask for up to `most` bytes of dynamic shared memory, once a device.  The limit is the kernel's, not a launch's: `most` is what any launch of it may need, so that a
// call of another thread never lowers it between this one's and its launch.
inline int pe_allow_smem(const void* kernel, int most, bool (&done)[64]) {
    int dev = 0;
    PE_TRY(cudaGetDevice(&dev));
    if (dev < 64 && done[dev]) return 0;
    PE_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    if (dev < 64) done[dev] = true;
    return 0;
}

inline int& pe_pdl_enabled() { static int on = 1; return on; }

template <typename... KArgs, typename... Args>
inline cudaError_t pe_launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                             Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pe_pdl_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

// The same with the CTAs of `cluster_x` consecutive blockIdx.x forming one thread-block cluster.
template <typename... KArgs, typename... Args>
inline cudaError_t pe_launch_cluster(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                                     unsigned cluster_x, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (pe_pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    if (cluster_x > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster_x; attr[n].val.clusterDim.y = 1; attr[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16_rn(v); }

// A vector of a norm weight or bias may be stored in either dtype.
__device__ __forceinline__ float load_as_f(const void* p, int dtype, size_t i) {
    return dtype == PE_F32 ? ((const float*)p)[i] : __bfloat162float(((const bf16*)p)[i]);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Block-wide sum, the same value returned to every thread.  `scratch` holds 33 floats.
// The order of additions depends on the block size only, never on the data.
__device__ __forceinline__ float block_sum(float v, float* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = (blockDim.x + 31) >> 5;
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) scratch[warp] = v;
    __syncthreads();
    if (warp == 0) {
        float t = lane < nwarps ? scratch[lane] : 0.f;
        t = warp_sum(t);
        if (lane == 0) scratch[32] = t;
    }
    __syncthreads();
    return scratch[32];
}
__device__ __forceinline__ float block_max(float v, float* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = (blockDim.x + 31) >> 5;
    v = warp_max(v);
    __syncthreads();
    if (lane == 0) scratch[warp] = v;
    __syncthreads();
    if (warp == 0) {
        float t = lane < nwarps ? scratch[lane] : -INFINITY;
        t = warp_max(t);
        if (lane == 0) scratch[32] = t;
    }
    __syncthreads();
    return scratch[32];
}
