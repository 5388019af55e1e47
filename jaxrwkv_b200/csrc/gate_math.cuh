// Logistic functions and pairs of floats for the elementwise operators.
#pragma once
#include "common.cuh"

namespace b200wkv {

// The hardware's exponential and reciprocal (2 and 1 units in the last place, results below 2^-126 are 0).
__device__ __forceinline__ float ex2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// min that keeps what is no number
__device__ __forceinline__ float min_nan(float x, float y) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}

// max that keeps what is no number
__device__ __forceinline__ float max_nan(float x, float y) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}

// Two numbers in one instruction: these kernels are short of issue slots before anything else.  They stay in one 64-bit register
// from instruction to instruction; as two 32-bit values they would be moved together and apart around each.
struct F2 { unsigned long long v; };
__device__ __forceinline__ F2 make_f2(float x, float y) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 parts(F2 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 both(float x) { return make_f2(x, x); }
// two adjacent elements
__device__ __forceinline__ F2 unpack_pair(uint32_t q) { return make_f2(__uint_as_float(q << 16), __uint_as_float(q & 0xffff0000u)); }

// p = sigmoid(z) and q = 1 - p = p e^-z, both to full relative precision.  The exponential is kept below 2^126, so that neither factor
// leaves the range (p is at least 2^-126 then, and not 0); kBounded: z is -87 or more, so it is.  For bf16 streams by the hardware's
// exponential, whose argument's rounding is 2^-24 |z| at most; the reciprocal is the hardware's in both types.
template <typename T, bool kBounded = false> __device__ __forceinline__ void sigmoid_pair(F2 z, F2& p, F2& q) {
    F2 e;
    if constexpr (sizeof(T) == 4) {
        const float2 t = parts(z);
        e = kBounded ? make_f2(expf(-t.x), expf(-t.y)) : make_f2(expf(min_nan(-t.x, 87.f)), expf(min_nan(-t.y, 87.f)));
    } else {
        const float2 t = parts(mul2(z, both(-1.44269504f)));
        e = kBounded ? make_f2(ex2_approx(t.x), ex2_approx(t.y)) : make_f2(ex2_approx(min_nan(t.x, 126.f)), ex2_approx(min_nan(t.y, 126.f)));
    }
    const float2 d = parts(add2(e, both(1.f)));
    p = make_f2(rcp_approx(d.x), rcp_approx(d.y));
    q = mul2(e, p);
}

}  // namespace b200wkv
