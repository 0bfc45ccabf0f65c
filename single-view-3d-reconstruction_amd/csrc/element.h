// Element types of the layer norm and optimizer kernels: fp32 in registers, fp32 / fp16 / bf16 in memory.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sv3d_hip.h"

namespace sv3d {

using f16 = _Float16;
using bf16 = __bf16;

// to_float is exact; from_float rounds to nearest even (at most half a step: 2^-11 of the value for fp16,
// 2^-8 for bf16)
template <class T>
__device__ inline float to_float(T v) { return (float)v; }
template <class T>
__device__ inline T from_float(float v) { return (T)v; }

inline bool known_type(int32_t t) { return t == SV3D_F32 || t == SV3D_F16 || t == SV3D_BF16; }
inline int type_bytes(int32_t t) { return t == SV3D_F32 ? 4 : 2; }
inline bool aligned(const void *p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

inline int launch_status() { return hipGetLastError() == hipSuccess ? SV3D_OK : SV3D_ERR_LAUNCH; }

}  // namespace sv3d
