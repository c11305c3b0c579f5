// Shared device helpers of the sequence operators (layer_norm.hip, gru_scan.hip, gated_mlp.hip): element types and their vectors.
// These files are compiled without packed fp32 instructions (build.py), see MOTIF_SCALAR_F32 in common.h.
#pragma once
#include <type_traits>
#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// Calls f with a null pointer of the element type that `dtype` names; false for an unknown code.
template <typename F>
static inline bool seq_dispatch(int dtype, F&& f) {
    switch (dtype) {
        case MOTIF_F32: f((float*)nullptr); return true;
        case MOTIF_BF16: f((bf16_t*)nullptr); return true;
        case MOTIF_F16: f((f16_t*)nullptr); return true;
        default: return false;
    }
}
static inline int seq_size(int dtype) { return dtype == MOTIF_F32 ? 4 : 2; }
static inline bool seq_dtype_ok(int dtype) { return dtype == MOTIF_F32 || dtype == MOTIF_BF16 || dtype == MOTIF_F16; }
// A null pointer counts as aligned.
static inline bool seq_aligned(const void* p, int bytes) { return ((unsigned long long)p & (unsigned long long)(bytes - 1)) == 0; }

template <typename T, int N>
struct alignas(sizeof(T) * N) SeqVec { T v[N]; };

template <typename T, int N>
__device__ __forceinline__ void seq_load(const T* p, float (&out)[N]) {
    const SeqVec<T, N> x = *(const SeqVec<T, N>*)p;
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = (float)x.v[i];
}
template <typename T, int N>
__device__ __forceinline__ void seq_store(T* p, const float (&in)[N]) {
    SeqVec<T, N> x;
#pragma unroll
    for (int i = 0; i < N; ++i) x.v[i] = (T)in[i];
    *(SeqVec<T, N>*)p = x;
}
// N values from an address that is a multiple of 16 bytes, or of their whole size where that is less.
template <typename T, int N>
__device__ __forceinline__ void seq_load16(const T* p, float (&out)[N]) {
    constexpr int P = 16 / (int)sizeof(T) < N ? 16 / (int)sizeof(T) : N;
#pragma unroll
    for (int j = 0; j < N; j += P) {
        const SeqVec<T, P> x = *(const SeqVec<T, P>*)(p + j);
#pragma unroll
        for (int i = 0; i < P; ++i) out[j + i] = (float)x.v[i];
    }
}
template <typename T, int N>
__device__ __forceinline__ void seq_store16(T* p, const float (&in)[N]) {
    constexpr int P = 16 / (int)sizeof(T) < N ? 16 / (int)sizeof(T) : N;
#pragma unroll
    for (int j = 0; j < N; j += P) {
        SeqVec<T, P> x;
#pragma unroll
        for (int i = 0; i < P; ++i) x.v[i] = (T)in[j + i];
        *(SeqVec<T, P>*)(p + j) = x;
    }
}
template <int N>
__device__ __forceinline__ void seq_param_vec(const void* p, long i, int dtype, float (&out)[N]) {
    if (dtype == MOTIF_F32) seq_load16<float, N>((const float*)p + i, out);
    else if (dtype == MOTIF_BF16) seq_load16<bf16_t, N>((const bf16_t*)p + i, out);
    else seq_load16<f16_t, N>((const f16_t*)p + i, out);
}
// One value of a parameter whose type is not the data's (uniform branch).
__device__ __forceinline__ float seq_param(const void* p, long i, int dtype) {
    return dtype == MOTIF_F32 ? ((const float*)p)[i] : dtype == MOTIF_BF16 ? (float)((const bf16_t*)p)[i] : (float)((const f16_t*)p)[i];
}
__device__ __forceinline__ void seq_param_store(void* p, long i, int dtype, float v) {
    if (dtype == MOTIF_F32) ((float*)p)[i] = v;
    else if (dtype == MOTIF_BF16) ((bf16_t*)p)[i] = (bf16_t)v;
    else ((f16_t*)p)[i] = (f16_t)v;
}

// layer_norm.hip: out0[c] = sum over the nb rows of part [nb][2 D] of column c, out1[c] of column D + c (either may be null), fixed order.
int seq_colsum2(const float* part, int nb, long D, void* out0, void* out1, int dtype, hipStream_t s);
