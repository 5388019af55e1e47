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

// Two numbers in one instruction: these kernels are short of issue slots before anything else.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// two adjacent elements
__device__ __forceinline__ float2 unpack_pair(uint32_t q) { return make_float2(__uint_as_float(q << 16), __uint_as_float(q & 0xffff0000u)); }

// p = sigmoid(z) and q = 1 - p = p e^-z, both to full relative precision.  The exponential is kept below 2^126, so that neither factor
// leaves the range (p is at least 2^-126 then, and not 0).  For bf16 streams by the hardware's exponential, whose argument's
// rounding is 2^-24 |z| at most.
template <typename T> __device__ __forceinline__ void sigmoid_pair(float2 z, float2& p, float2& q) {
    float2 e;
    if constexpr (sizeof(T) == 4) {
        e = make_float2(expf(min_nan(-z.x, 87.f)), expf(min_nan(-z.y, 87.f)));
    } else {
        const float2 t = mul2(z, both(-1.44269504f));
        e = make_float2(ex2_approx(min_nan(t.x, 126.f)), ex2_approx(min_nan(t.y, 126.f)));
    }
    const float2 d = add2(e, both(1.f));
    p = make_float2(rcp_approx(d.x), rcp_approx(d.y));
    q = mul2(e, p);
}

}  // namespace b200wkv
