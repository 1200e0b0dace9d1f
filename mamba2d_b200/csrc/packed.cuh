// fp32 values in pairs, whose sums and products are one instruction.
#pragma once

#include <cuda_runtime.h>

namespace m2d {

// One value or two: packed arithmetic for two.  Single ones are rounded where those are.
template <int VEC> struct Num;
template <> struct Num<1> {
    float v;
    __device__ __forceinline__ static Num all(float f) { return {f}; }
    __device__ __forceinline__ float get(int) const { return v; }
    __device__ __forceinline__ void set(int, float f) { v = f; }
};
template <> struct Num<2> {
    unsigned long long v;
    __device__ __forceinline__ static Num make(float a, float b) {
        Num r;
        asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
        return r;
    }
    __device__ __forceinline__ static Num all(float f) { return make(f, f); }
    __device__ __forceinline__ float get(int i) const {
        float a, b;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
        return i ? b : a;
    }
    __device__ __forceinline__ void set(int i, float f) { *this = i ? make(get(0), f) : make(f, get(1)); }
};
__device__ __forceinline__ Num<1> fma_(Num<1> a, Num<1> b, Num<1> c) { return {fmaf(a.v, b.v, c.v)}; }
__device__ __forceinline__ Num<1> mul_(Num<1> a, Num<1> b) { return {__fmul_rn(a.v, b.v)}; }
__device__ __forceinline__ Num<1> add_(Num<1> a, Num<1> b) { return {__fadd_rn(a.v, b.v)}; }
__device__ __forceinline__ Num<2> fma_(Num<2> a, Num<2> b, Num<2> c) {
    Num<2> r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ Num<2> mul_(Num<2> a, Num<2> b) {
    Num<2> r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Num<2> add_(Num<2> a, Num<2> b) {
    Num<2> r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
template <int VEC> __device__ __forceinline__ Num<VEC> neg_(Num<VEC> a) { return mul_(a, Num<VEC>::all(-1.f)); }

}  // namespace m2d
