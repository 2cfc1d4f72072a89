// What the small kernels around the packed linears share: conversions, the prologue and the launch of programmatic
// dependent launch.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "kernels.h"

namespace mg {

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The rotation with its roundings spelled out: left to the compiler, the kernels that rotate contracted the same expression
// differently, and a model whose layers amplify one flipped bit showed it.
__device__ __forceinline__ float rotated_even(float a, float c, float cs, float sn) { return __fmaf_rn(a, cs, -__fmul_rn(c, sn)); }
__device__ __forceinline__ float rotated_odd(float a, float c, float cs, float sn) { return __fmaf_rn(c, cs, __fmul_rn(a, sn)); }

// Programmatic dependent launch: let the next kernel of the stream start its prologue now (the packed products
// prefetch their weights there), then wait until the previous kernel's results are complete and visible.  Both
// are no-ops for a kernel that was launched without the attribute and has no dependents.
__device__ __forceinline__ void pdl_prologue() {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <typename Kernel, typename... Args>
static int launch_helper(Kernel kernel, dim3 grid, unsigned block, cudaStream_t stream, bool pdl, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  if (pdl) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? MG_OK : MG_ERR_CUDA;
}

}  // namespace mg
