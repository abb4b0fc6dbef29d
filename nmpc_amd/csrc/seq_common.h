// Element types and small helpers of the sequence operators (seq_conv.hip, seq_scan.hip, seq_ffn.hip).
#pragma once
#include "../../include/nmpc_amd.h"
#include "common.h"

namespace nmpc {

typedef __bf16 bf16;
typedef _Float16 f16;

// V neighbouring elements moved as one access (V * sizeof(T) = 16 bytes in the vector paths, one element otherwise)
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T v[V];
};
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
    return *reinterpret_cast<const Vec<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, V>& x) {
    *reinterpret_cast<Vec<T, V>*>(p) = x;
}

constexpr float LOG2E = 1.44269504088896340736f;

// 1 / (1 + e^-x), exponential and reciprocal of one unit in the last place each; e^-x overflows to infinity and the reciprocal to 0 where the value is below 2^-126
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-LOG2E * x)); }

// steps of sequence b that count: lengths[b] clamped to 0 .. L
__device__ __forceinline__ int seq_length(const int* lengths, int b, int L) {
    if (!lengths) return L;
    const int n = lengths[b];
    return n < 0 ? 0 : (n > L ? L : n);
}

// host: may V-element accesses be used on a tensor with these strides (in elements)?
template <typename T>
inline bool vec_ok(const void* p, long long s0, long long s1, int V) {
    return !p || ((reinterpret_cast<uintptr_t>(p) % (V * sizeof(T))) == 0 && s0 % V == 0 && s1 % V == 0);
}

}  // namespace nmpc

// runs its last argument with the element type bound to T_
#define NMPC_DTYPE_SWITCH(dtype, ...)                                       \
    switch (dtype) {                                                        \
        case NMPC_F32: { using T_ = float; __VA_ARGS__ } break;                    \
        case NMPC_BF16: { using T_ = nmpc::bf16; __VA_ARGS__ } break;              \
        case NMPC_F16: { using T_ = nmpc::f16; __VA_ARGS__ } break;                \
        default: nmpc::set_error("unknown element type %d", dtype); return 1; \
    }
