// sx_two.cuh — 32-bit arithmetic two values at a time (sm_100a has it as one instruction).
#pragma once

#include <stdint.h>

namespace sx {
namespace tc {

// Two 32-bit values that one instruction works on.
struct Two {
    uint64_t v;
};
__device__ __forceinline__ Two two(float lo, float hi) {
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void split(Two x, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x.v)); }
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

}  // namespace tc
}  // namespace sx
