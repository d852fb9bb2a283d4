// Shared by the token operators (wst_tokens.hip, wst_attention.hip): element types, unaligned vector access, wave and
// block sums, the error string, launch checks.
#ifndef WST_TOKENS_H
#define WST_TOKENS_H

#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstdio>

#include "wst_hip.h"

namespace wst_tok {

using bf16 = __bf16;
using f16 = _Float16;

// Sets the thread's error text (wst_tokens_last_error) and returns `code`. Nothing here allocates or throws.
__attribute__((visibility("hidden"))) int fail(int code, const char* fmt, ...);
// Status of the launches just made.
__attribute__((visibility("hidden"))) int launched(const char* what);

template <typename T, int N>
struct Vec {
    T v[N];
};

// N elements from / to a pointer that is aligned to one element only: the compiler emits wide accesses, which global
// memory takes at any alignment; rows of odd lengths then need no path of their own.
template <int N, typename T>
__device__ __forceinline__ void load(const T* p, float (&out)[N]) {
    Vec<T, N> t;
    __builtin_memcpy(&t, p, sizeof(t));
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = static_cast<float>(t.v[i]);
}
template <int N, typename T>
__device__ __forceinline__ void store(T* p, const float (&in)[N]) {
    Vec<T, N> t;
#pragma unroll
    for (int i = 0; i < N; ++i) t.v[i] = static_cast<T>(in[i]);   // to nearest, ties to even
    __builtin_memcpy(p, &t, sizeof(t));
}

// Value i of an array whose type is known at run time only (weights, biases): a uniform branch.
__device__ __forceinline__ float load_as(const void* p, int dtype, int64_t i) {
    if (dtype == WST_F32) return static_cast<const float*>(p)[i];
    if (dtype == WST_BF16) return static_cast<float>(static_cast<const bf16*>(p)[i]);
    return static_cast<float>(static_cast<const f16*>(p)[i]);
}
__device__ __forceinline__ void store_as(void* p, int dtype, int64_t i, float v) {
    if (dtype == WST_F32) static_cast<float*>(p)[i] = v;
    else if (dtype == WST_BF16) static_cast<bf16*>(p)[i] = static_cast<bf16>(v);
    else static_cast<f16*>(p)[i] = static_cast<f16>(v);
}
template <int N>
__device__ __forceinline__ void load_as_n(const void* p, int dtype, int64_t i, float (&out)[N]) {
    if (dtype == WST_F32) load<N>(static_cast<const float*>(p) + i, out);
    else if (dtype == WST_BF16) load<N>(static_cast<const bf16*>(p) + i, out);
    else load<N>(static_cast<const f16*>(p) + i, out);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}

}  // namespace wst_tok

#endif  // WST_TOKENS_H
