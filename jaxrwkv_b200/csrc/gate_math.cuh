// Exponentials and logistic functions of the elementwise operators, by the element type that their results go to.
#pragma once
#include "common.cuh"

namespace b200wkv {

// bf16 results carry 8 bits: the hardware's exponential and quotient (a few units of 2^-23) are far below their rounding.
template <typename T> __device__ __forceinline__ float exp_of(float x) { return sizeof(T) == 4 ? expf(x) : __expf(x); }
template <typename T> __device__ __forceinline__ float inverse(float x) { return sizeof(T) == 4 ? 1.f / x : __fdividef(1.f, x); }

// p = sigmoid(z) and q = 1 - p, both to full relative precision: with t = e^-|z| the larger is 1 / (1 + t), the smaller t times that.
template <typename T> __device__ __forceinline__ void sigmoid_pair(float z, float& p, float& q) {
    const float t = exp_of<T>(-fabsf(z)), big = inverse<T>(1.f + t), small = t * big;
    p = z >= 0.f ? big : small;
    q = z >= 0.f ? small : big;
}

}  // namespace b200wkv
