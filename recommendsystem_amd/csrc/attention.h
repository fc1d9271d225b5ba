// What the attention kernels share: their arguments, the mask, and how rows are read and written.
#pragma once
#include "lowp.h"

struct AttnOperand {
    const void* p;
    long long b, t, h;      // strides in elements
};

struct AttnArgs {
    AttnOperand q, k, v, o, go;              // go: gradient of o
    void *out, *dq, *dk, *dv;                // contiguous
    float *lse, *delta;                      // [B, Hq, Tq]
    const int *len, *qlen, *qstart;          // [B] or null
    int B, Tq, Tk, Hk, G, D, causal, start;
    float scale;
    int tiles, splits;                       // row (key) tiles per (sample, key head); shares of the keys (rows)
    int dealt;                               // order of the workgroups: pairs (samples) dealt out at a time, 0: in runs
    // with splits > 1: forward [splits, B * Hk, Tq * G, D] and lse in base 2 [.., Tq * G], dk / dv [splits, 2, B, Tk, Hk, D]
    float *part_o, *part_ml;
    int vec;                                 // 16-byte loads from q, k, v, o, go
    int out_vec;                             // four elements at once to the outputs
};

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

typedef short rs_s16x4 __attribute__((ext_vector_type(4)));

// E elements from column col of a row of D (zeros behind D, and everywhere when the row has no part).
template <typename T, bool VEC> __device__ __forceinline__ typename RsVec<T>::V fetch(const T* row, int col, int D, bool live) {
    typename RsVec<T>::V r;
    constexpr int E = RsVec<T>::E;
#pragma unroll
    for (int e = 0; e < E; ++e) r[e] = (T)0.f;
    if (live && col < D) {
        if constexpr (VEC) {
            r = *(const typename RsVec<T>::V*)(row + col);
        } else if (col + E <= D) {
            r = *(const typename RsVec<T>::U*)(row + col);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (col + e < D) r[e] = row[col + e];
        }
    }
    return r;
}

// A fragment that was loaded in front of a loop has arrived: without a use there, the wait for it would stand in the loop
// and hold up the asynchronous loads, too.
template <typename V> __device__ __forceinline__ void settle(V& v) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    union { V v; u32x4 u; } x;
    x.v = v;
    asm volatile("" : "+v"(x.u));
    v = x.v;
}
// What a lane's row sees: keys below the result.
__device__ __forceinline__ int row_limit(const AttnArgs& a, int b, int i) {
    int lim = a.len ? min(max(a.len[b], 0), a.Tk) : a.Tk;
    const int rows = a.qlen ? min(a.qlen[b], a.Tq) : a.Tq;
    if (i >= rows) return 0;
    if (a.causal) {
        const long long last = (long long)i + (a.qstart ? a.qstart[b] : a.start) + 1;
        lim = last < lim ? (last < 0 ? 0 : (int)last) : lim;
    }
    return lim;
}

// fp16's range.  P lies in 0..1 and dS is as small as the gradients of o, while fp16 loses bits below 2^-14 and everything below
// 2^-25; the sums over keys or rows are larger and would keep what the terms lost.  So P is made 2^8 times as large, a shift
// of the exponent that exp2 gets and no instruction of its own (elements down to 2^-22 keep all their bits; more of a shift
// would overflow for rows whose huge scores, of 10^7 and up, leave exp2 an argument off by several ones), and dS is
// multiplied by a power of two that follows its largest element.  Both are taken out in fp32 behind the sums.  Gradients
// of 1e-4 over 2048 keys were 4.1 (heads of 128) and 5.7 times (64) as far off as one final rounding without this, and are 1.0
// times with it; 2 x 8192 causal, 16 heads of 128: forward 613 us as before, dq 806 -> 850, dk / dv 1233 -> 1345 (side by side).
template <typename T> constexpr float P_SHIFT = 0.f;
template <typename T> constexpr float P_UNIT = 1.f;
template <> constexpr float P_SHIFT<_Float16> = 8.f;
template <> constexpr float P_UNIT<_Float16> = 1.f / 256;

// The factor 2^exp of the dS that are summed together.  The largest element gets to 2^12..2^13 and may grow to 2^15 before
// the factor falls: elements down to 2^-26 of the largest one keep all their bits.
struct Range {
    float most = 0.f;        // 0 until an element was seen
    int exp = 0;
    __device__ __forceinline__ bool past(float top) const { return top > most; }      // top: scaled by the present factor
    // the exponent to add
    __device__ __forceinline__ int follow(float top) {
        if (!past(top)) return 0;
        const int by = max(-100, min(12 + 127 - (int)(__float_as_uint(top) >> 23), 60 - exp));
        exp += by;
        most = 32768.f;
        return by;
    }
    __device__ __forceinline__ float unit() const { return ldexpf(1.f, -exp); }
};

// A row's lse for the backward, in base 2.  -inf: the row sees nothing, or its scores all overflowed to -inf (fp32 operands
// near 1e20); it got zeros, and exp2(z - inf) = 0 gives it no part in any gradient.
__device__ __forceinline__ float back_lse(float lse) { return lse == -INFINITY ? INFINITY : lse * LOG2E; }

template <typename T> __device__ __forceinline__ const T* row_ptr(const AttnOperand& x, int b, int t, int h) {
    return (const T*)x.p + b * x.b + t * x.t + h * x.h;
}

// Four consecutive elements of an output row.
template <typename T> __device__ __forceinline__ void store4(T* row, int d, int D, bool vec, const float* v) {
    if (vec && d + 4 <= D) {
        if constexpr (sizeof(T) == 4) {
            *(rs_f32x4*)(row + d) = rs_f32x4{v[0], v[1], v[2], v[3]};
        } else {
            typedef T T4 __attribute__((ext_vector_type(4)));
            *(T4*)(row + d) = T4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < D) row[d + e] = (T)v[e];
    }
}

// 16x16 tiles: CK elements of the contraction in a fragment pair, 16 bytes a lane; lane l holds row (column) l % 16 and
// elements E (l / 16) .. of the CK.  A result holds column l % 16 and rows 4 (l / 16) + 0..3.
template <typename T> struct Mma16;
template <> struct Mma16<float> {
    static constexpr int CK = 16, E = 4, TILES = 1;          // TILES: row tiles that one contraction step over rows covers
    typedef rs_f32x4 V;
    static __device__ __forceinline__ rs_f32x4 mul(V a, V b, rs_f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};
template <> struct Mma16<__bf16> {
    static constexpr int CK = 32, E = 8, TILES = 2;
    typedef rs_bf16x8 V;
    static __device__ __forceinline__ rs_f32x4 mul(V a, V b, rs_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mma16<_Float16> {
    static constexpr int CK = 32, E = 8, TILES = 2;
    typedef rs_f16x8 V;
    static __device__ __forceinline__ rs_f32x4 mul(V a, V b, rs_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

// Over the four lanes that hold a column.
__device__ __forceinline__ float col_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float col_sum(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}

}  // namespace

// Few keys (attention_small.hip): whether a call is for these kernels, and the two directions.
bool rs_attention_small_ok(int dtype, int Tq, int Tk, int D);
int rs_attention_small_fwd(int dtype, const AttnArgs& a, hipStream_t stream);
int rs_attention_small_bwd(int dtype, const AttnArgs& a, hipStream_t stream);
