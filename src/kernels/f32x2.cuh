// Two float32 operations in one instruction (sm_100): half the issue slots of the same work in single ones.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace mgk {
namespace f32x2 {

struct Pair {
    float x, y;
};
__device__ __forceinline__ Pair both(float x) { return {x, x}; }

__device__ __forceinline__ Pair mul(Pair a, Pair b) {
    Pair d;
    asm("{\n .reg .b64 p, q, r;\n mov.b64 p, {%2, %3};\n mov.b64 q, {%4, %5};\n mul.rn.f32x2 r, p, q;\n mov.b64 {%0, %1}, r;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// (a sum of paired products comes out contracted into fused multiply-adds: where each is to be rounded on its
// own, the sums are single ones)
__device__ __forceinline__ Pair add(Pair a, Pair b) {
    Pair d;
    asm("{\n .reg .b64 p, q, r;\n mov.b64 p, {%2, %3};\n mov.b64 q, {%4, %5};\n add.rn.f32x2 r, p, q;\n mov.b64 {%0, %1}, r;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
    Pair d;
    asm("{\n .reg .b64 p, q, r, s;\n mov.b64 p, {%2, %3};\n mov.b64 q, {%4, %5};\n mov.b64 r, {%6, %7};\n"
        " fma.rn.f32x2 s, p, q, r;\n mov.b64 {%0, %1}, s;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

// the largest of three; a NaN is kept
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

}  // namespace f32x2
}  // namespace mgk
