// Element types of the sequence operators: fp32, bf16 and fp16 in memory, fp32 in registers.
#pragma once
#include "common.h"

enum { RS_F32 = 0, RS_BF16 = 1, RS_F16 = 2 };

typedef float rs_f32x4 __attribute__((ext_vector_type(4)));
typedef float rs_f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 rs_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 rs_f16x8 __attribute__((ext_vector_type(8)));

// V = the 16-byte vector of T, U = the same at any address, E = its elements.
template <typename T> struct RsVec;
template <> struct RsVec<float> {
    typedef rs_f32x4 V;
    typedef rs_f32x4 U __attribute__((aligned(4)));
    static constexpr int E = 4;
};
template <> struct RsVec<__bf16> {
    typedef rs_bf16x8 V;
    typedef rs_bf16x8 U __attribute__((aligned(2)));
    static constexpr int E = 8;
};
template <> struct RsVec<_Float16> {
    typedef rs_f16x8 V;
    typedef rs_f16x8 U __attribute__((aligned(2)));
    static constexpr int E = 8;
};

// E consecutive elements as fp32, in one 16-byte access.  WHOLE: p is aligned to 16 bytes and all E elements are there; else
// p is any element and the first `left` of E belong to the row (zeros for the others).  Stores round to nearest even once.
template <typename T, bool WHOLE> __device__ __forceinline__ void rs_load(const T* p, int left, float* v) {
    constexpr int E = RsVec<T>::E;
    if (WHOLE || left >= E) {
        typename RsVec<T>::V x;
        if constexpr (WHOLE) x = *(const typename RsVec<T>::V*)p;
        else x = *(const typename RsVec<T>::U*)p;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = (float)x[e];
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = e < left ? (float)p[e] : 0.f;
    }
}
template <typename T, bool WHOLE> __device__ __forceinline__ void rs_store(T* p, int left, const float* v) {
    constexpr int E = RsVec<T>::E;
    if (WHOLE || left >= E) {
        typename RsVec<T>::V x;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = (T)v[e];
        if constexpr (WHOLE) *(typename RsVec<T>::V*)p = x;
        else *(typename RsVec<T>::U*)p = x;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e < left) p[e] = (T)v[e];
    }
}

// Any number of workgroups: kernels launched so take rs_block_id() for their number and leave when it is past the last one.
// A grid dimension holds fewer than 2^32 lanes, which 2^21 workgroups of up to 1024 keep.
static inline dim3 rs_grid(long long blocks) {
    const long long x = blocks < (1 << 21) ? blocks : (1 << 21);
    return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}
__device__ __forceinline__ long long rs_block_id() { return (long long)blockIdx.y * gridDim.x + blockIdx.x; }

static inline int rs_elem_bytes(int dtype) { return dtype == RS_F32 ? 4 : 2; }
static inline bool rs_aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
