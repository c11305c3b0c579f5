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

// N values of T as they lie in memory, at any address that is a multiple of T's size: global memory takes 16-byte accesses at such addresses, so rows of
// any length and offset are read in 16-byte pieces (a lane whose piece would pass the row's end takes the last N values instead).
template <typename T, int N>
struct SeqRaw {
    T v[N];
    __device__ __forceinline__ float operator[](int i) const { return (float)v[i]; }
};
template <int BYTES> struct SeqWords { typedef unsigned type __attribute__((ext_vector_type(BYTES / 4))); };
template <> struct SeqWords<4> { typedef unsigned type; };
template <> struct SeqWords<2> { typedef unsigned short type; };

template <typename T, int N>
__device__ __forceinline__ SeqRaw<T, N> seq_raw(const T* p) {
    constexpr int B = sizeof(T) * N, P = B < 16 ? B : 16;
    typedef typename SeqWords<P>::type W;
    struct { W w[B / P]; } x;
#pragma unroll
    for (int i = 0; i < B / P; ++i) __builtin_memcpy(&x.w[i], (const char*)p + i * P, P);
    return __builtin_bit_cast(SeqRaw<T, N>, x);
}
// Keeps what was read as it was read: without this the compiler holds the fp32 values of the first walk for the second one, twice the registers.
template <typename T, int V>
__device__ __forceinline__ void seq_hold(SeqRaw<T, V>& x) {
    constexpr int B = sizeof(T) * V, P = B < 16 ? B : 16;
    static_assert(B == P, "");
    auto w = __builtin_bit_cast(typename SeqWords<P>::type, x);
    asm volatile("" : "+v"(w));
    x = __builtin_bit_cast(SeqRaw<T, V>, w);
}
template <typename T, int N>
__device__ __forceinline__ void seq_load(const T* p, float (&out)[N]) {
    const SeqRaw<T, N> x = seq_raw<T, N>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = x[i];
}
// `stream`: past the caches, for outputs that they would not hold until they are read (kSeqStream bytes and more).
constexpr long kSeqStream = 96L << 20;
template <typename T, int N>
__device__ __forceinline__ void seq_store(T* p, const float (&in)[N], bool stream = false) {
    constexpr int B = sizeof(T) * N, P = B < 16 ? B : 16;
    typedef typename SeqWords<P>::type W;
    typedef W __attribute__((aligned(sizeof(T)))) AnyW;
    SeqRaw<T, N> x;
#pragma unroll
    for (int i = 0; i < N; ++i) x.v[i] = (T)in[i];
    struct Words { W w[B / P]; };
    const Words y = __builtin_bit_cast(Words, x);
#pragma unroll
    for (int i = 0; i < B / P; ++i) {
        if (stream) __builtin_nontemporal_store(y.w[i], (AnyW*)((char*)p + i * P));
        else __builtin_memcpy((char*)p + i * P, &y.w[i], P);
    }
}
template <int N>
__device__ __forceinline__ void seq_param_vec(const void* p, long i, int dtype, float (&out)[N]) {
    if (dtype == MOTIF_F32) seq_load<float, N>((const float*)p + i, out);
    else if (dtype == MOTIF_BF16) seq_load<bf16_t, N>((const bf16_t*)p + i, out);
    else seq_load<f16_t, N>((const f16_t*)p + i, out);
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
