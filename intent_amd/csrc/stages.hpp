// What kernels share whose tiles pass the LDS in stages that are on their way while earlier ones are used, for gfx950.
#pragma once

#include "common.hpp"

namespace intent_hip {
namespace {

typedef __attribute__((address_space(3))) void lds_void_t;

// s_waitcnt with only the vector-memory counter constrained (vmcnt <= n).
#define INTENT_WAIT_VMCNT(n) __builtin_amdgcn_s_waitcnt((((n) & 0xF) | (((n) >> 4) << 14) | (0x7 << 4) | (0xF << 8)))

// s_barrier with an acquire fence alone: a release fence would wait for every load into the LDS that is on its way.
__device__ __forceinline__ void stage_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  __builtin_amdgcn_sched_barrier(0);
}

// What a lane loads that has nothing to load: behind K, or behind the last token.
__device__ const uint4 kZeroUnit = {0u, 0u, 0u, 0u};

}  // namespace
}  // namespace intent_hip
