// gw_learn.hpp — what the policy operators' translation units share: errors,
// element types, wave reductions (gw_policy.hip, gw_recurrence.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/gw_learn.h"

#define WAVE 64

// gw_learn_last_error's text (this thread's)
void gw_learn_set_err(const char* fmt, ...);

#define LEARN_NEED(cond, ...)                    \
    do {                                         \
        if (!(cond)) {                           \
            gw_learn_set_err(__VA_ARGS__);       \
            return GW_E_INVALID;                 \
        }                                        \
    } while (0)

#define LEARN_LAUNCHED()                                                        \
    do {                                                                        \
        const hipError_t e_ = hipGetLastError();                                \
        if (e_ != hipSuccess) {                                                 \
            gw_learn_set_err("%s: %s", __func__, hipGetErrorString(e_));        \
            return GW_E_HIP;                                                    \
        }                                                                       \
    } while (0)

namespace {

typedef _Float16 f16;
typedef __bf16 bf16;

constexpr float NEG_INF = -__builtin_inff();

// the larger of two, NaN if either is: a NaN logit must not vanish in a maximum
__device__ __forceinline__ float max_nan(float a, float b) { return (b > a || b != b) ? b : a; }

// what a wave's lanes have written to LDS is there for its other lanes
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <class V>
__device__ __forceinline__ V wave_sum(V v)
{
#pragma unroll
    for (int o = WAVE / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

__device__ __forceinline__ float wave_max_nan(float v)
{
#pragma unroll
    for (int o = WAVE / 2; o > 0; o >>= 1) v = max_nan(v, __shfl_xor(v, o));
    return v;
}

}  // namespace
