// Rotary positions: of every head's first R of D elements, pair i -- elements (i, i + R/2), or neighbours (2i, 2i + 1) --
// is turned by the angle of its token's position:  (a, b) -> (a cos - b sin, b cos + a sin).  The rest is copied.  The
// inverse turns by the negative angle, which is also the way gradients go.
//
// cos and sin come from tables [P, R/2] the caller made once, in 64 bits, so that far positions keep their angles; the
// products are fp32 and rounded once.  Bound by memory: q and k are read and written once, in one launch; a lane takes
// one 16-byte vector (two of them when halves are paired) where R, D, the strides and the addresses allow, else one pair.
// The table's row of a token is shared by its heads and comes out of the caches.  16384 tokens of 40 heads of 128, half of each
// turned, bf16: 70 us a direction, 4.8 TB/s (a 4 GiB copy: 4.8).
#include "lowp.h"
#include "../../include/rs_hip.h"

#pragma clang fp contract(fast)

namespace {

constexpr int TOKENS_MAX = 8;      // tokens of a workgroup at most

struct RotaryArgs {
    const void *q, *k;
    long long qb, qt, qh, kb, kt, kh;      // strides in elements; outputs are contiguous
    int Hq, Hk, T, D, R;
    long long tokens;
    const void* pos;
    int pos64;
    long long pb, pt;
    const float *cos, *sin;
    int P;
    float sign;
    void *qo, *ko;
    int* err;
    int per_block;                         // tokens of a workgroup
};

// VE elements: an aligned 16-byte vector or one element.
template <typename T, int VE> __device__ __forceinline__ void load(const T* p, float* v) {
    if constexpr (VE == 1) v[0] = (float)*p;
    else rs_load<T, true>(p, VE, v);
}
template <typename T, int VE> __device__ __forceinline__ void store(T* p, const float* v) {
    if constexpr (VE == 1) *p = (T)v[0];
    else rs_store<T, true>(p, VE, v);
}

template <typename T, int VE, bool PAIRED>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
    __shared__ int s_pos[TOKENS_MAX];
    const long long token0 = rs_block_id() * a.per_block;
    if (threadIdx.x < a.per_block && token0 + threadIdx.x < a.tokens) {
        const long long tok = token0 + threadIdx.x, b = tok / a.T, t = tok - b * a.T;
        const long long at = b * a.pb + t * a.pt;
        long long p = a.pos64 ? ((const long long*)a.pos)[at] : (long long)((const int*)a.pos)[at];
        if (p < 0 || p >= a.P) {           // reads row 0, the caller finds the flag
            *a.err = 1;
            p = 0;
        }
        s_pos[threadIdx.x] = (int)p;
    }
    __syncthreads();
    const int half = a.R / 2, H = a.Hq + a.Hk;
    const unsigned turn = PAIRED ? (VE == 1 ? half : a.R / VE) : half / VE;     // units that turn, then units that copy
    const unsigned units = turn + (a.D - a.R) / VE;
    const unsigned items = units * H * a.per_block;
    for (unsigned it = threadIdx.x; it < items; it += 256) {
        const unsigned row = it / units, u = it - row * units, ti = row / H;
        const int h = row - ti * H;
        const long long tok = token0 + ti;
        if (tok >= a.tokens) return;
        const long long b = tok / a.T, t = tok - b * a.T;
        const bool is_q = h < a.Hq;
        const T* in = is_q ? (const T*)a.q + b * a.qb + t * a.qt + h * a.qh : (const T*)a.k + b * a.kb + t * a.kt + (h - a.Hq) * a.kh;
        T* out = is_q ? (T*)a.qo + (tok * a.Hq + h) * a.D : (T*)a.ko + (tok * a.Hk + (h - a.Hq)) * a.D;
        if (u >= turn) {
            const unsigned n = a.R + (u - turn) * VE;
            if constexpr (VE == 1) out[n] = in[n];
            else *(typename RsVec<T>::V*)(out + n) = *(const typename RsVec<T>::V*)(in + n);
            continue;
        }
        const float* cs = a.cos + (long long)s_pos[ti] * half;
        const float* sn = a.sin + (long long)s_pos[ti] * half;
        if constexpr (!PAIRED) {
            const unsigned n = u * VE;
            float x[VE], y[VE], p[VE], q[VE];
            load<T, VE>(in + n, x);
            load<T, VE>(in + half + n, y);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float c = cs[n + e], s = sn[n + e] * a.sign;
                p[e] = x[e] * c - y[e] * s;
                q[e] = y[e] * c + x[e] * s;
            }
            store<T, VE>(out + n, p);
            store<T, VE>(out + half + n, q);
        } else if constexpr (VE == 1) {
            const float x = (float)in[2 * u], y = (float)in[2 * u + 1], c = cs[u], s = sn[u] * a.sign;
            out[2 * u] = (T)(x * c - y * s);
            out[2 * u + 1] = (T)(y * c + x * s);
        } else {
            const unsigned n = u * VE;
            float x[VE];
            load<T, VE>(in + n, x);
#pragma unroll
            for (int e = 0; e < VE; e += 2) {
                const float c = cs[(n + e) / 2], s = sn[(n + e) / 2] * a.sign, v = x[e];
                x[e] = v * c - x[e + 1] * s;
                x[e + 1] = x[e + 1] * c + v * s;
            }
            store<T, VE>(out + n, x);
        }
    }
}

template <typename T> int launch(const RotaryArgs& a, bool vec, bool paired, hipStream_t stream) {
    constexpr int E = RsVec<T>::E;
    const dim3 grid = rs_grid(rs_cdiv(a.tokens, a.per_block));
    if (vec && paired) hipLaunchKernelGGL((rotary_kernel<T, E, true>), grid, dim3(256), 0, stream, a);
    else if (vec) hipLaunchKernelGGL((rotary_kernel<T, E, false>), grid, dim3(256), 0, stream, a);
    else if (paired) hipLaunchKernelGGL((rotary_kernel<T, 1, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((rotary_kernel<T, 1, false>), grid, dim3(256), 0, stream, a);
    RS_CHECK_LAUNCH("rs_rotary");
    return RS_OK;
}

}  // namespace

extern "C" int rs_rotary(int dtype, const void* q, long long qb, long long qt, long long qh, int Hq, const void* k, long long kb,
                         long long kt, long long kh, int Hk, int B, int T, int D, int R, int interleaved, const void* positions,
                         int positions_i64, long long pb, long long pt, const float* cos_table, const float* sin_table,
                         int max_positions, int inverse, void* q_out, void* k_out, int* err_flag, rs_stream_t stream) {
    RS_CHECK_ARG(dtype == RS_F32 || dtype == RS_BF16 || dtype == RS_F16, "rs_rotary: type %d not served", dtype);
    RS_CHECK_ARG(B >= 0 && T >= 0 && Hq >= 0 && Hk >= 0 && D > 0 && R > 0 && R <= D && R % 2 == 0 && max_positions > 0,
                 "rs_rotary: bad shape B=%d T=%d Hq=%d Hk=%d D=%d R=%d", B, T, Hq, Hk, D, R);
    const long long tokens = (long long)B * T;
    if (tokens == 0 || Hq + (long long)Hk == 0) return RS_OK;
    RS_CHECK_ARG((Hq + (long long)Hk) * D <= (1 << 24) && tokens <= 0x7fffffffLL, "rs_rotary: %lld tokens of %d x %d elements are too many", tokens,
                 Hq + Hk, D);
    RS_CHECK_ARG((Hq == 0 || (q && q_out)) && (Hk == 0 || (k && k_out)) && positions && cos_table && sin_table && err_flag,
                 "rs_rotary: null argument");
    const int e = 16 / rs_elem_bytes(dtype);
    // 16-byte accesses: every vector lies within one half, within the turned or the copied part, and starts at a
    // multiple of 16 bytes
    const bool vec = (interleaved ? R : R / 2) % e == 0 && D % e == 0 && (D - R) % e == 0 &&
                     (Hq == 0 || (rs_aligned16(q) && rs_aligned16(q_out) && qb % e == 0 && qt % e == 0 && qh % e == 0)) &&
                     (Hk == 0 || (rs_aligned16(k) && rs_aligned16(k_out) && kb % e == 0 && kt % e == 0 && kh % e == 0)) &&
                     rs_aligned16(cos_table) && rs_aligned16(sin_table);
    // a workgroup takes enough tokens to give each lane a few vectors, as long as there are workgroups for every CU
    const int per_token = (Hq + Hk) * (vec ? (interleaved ? D / e : (D - R / 2) / e) : D - R / 2);
    int per_block = 1;
    while (per_block < TOKENS_MAX && per_block * per_token < 512 && tokens / (2 * per_block) >= 1024) per_block *= 2;
    const RotaryArgs a = {q, k, qb, qt, qh, kb, kt, kh, Hq, Hk, T, D, R, tokens, positions, positions_i64, pb, pt, cos_table, sin_table,
                          max_positions, inverse ? -1.f : 1.f, q_out, k_out, err_flag, per_block};
    if (dtype == RS_F32) return launch<float>(a, vec, interleaved != 0, stream);
    if (dtype == RS_BF16) return launch<__bf16>(a, vec, interleaved != 0, stream);
    return launch<_Float16>(a, vec, interleaved != 0, stream);
}
