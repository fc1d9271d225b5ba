// Layer norm over the last dimension with an optional residual add in front, forward and backward, fp32 / bf16 / fp16:
//   s = round(x + r),  mean = avg(s),  rstd = 1 / sqrt(avg((s - mean)^2) + eps),  y = (s - mean) rstd w + b
//   xhat = (s - mean) rstd,  g = dy w,  dx = rstd (g - avg(g) - xhat avg(g xhat)) + ds,
//   dw = sum_rows dy xhat,  db = sum_rows dy
// All statistics and sums are fp32; the variance is that of the centred values (no E[x^2] - mean^2 cancellation).
//
// Both directions are bound by memory: a row is read once into registers by LPR lanes that own 16 elements each, as 16-byte
// vectors (WHOLE: aligned ones, where N, the strides and the addresses allow; else at any address, the row's last vector
// element by element), reduced across those lanes and written once.  LPR is the smallest of 8, 32, 64, 256 and 1024 that covers the row: rows of up to 1024 elements need no
// workgroup barrier, and a workgroup holds 256 / LPR rows at a time.  Rows beyond 16384 elements go through a
// workgroup of 1024 that reads them again from the caches for each pass.
//
// The backward's workgroups walk over the rows in steps of the grid, so a lane meets the same columns in every row and
// keeps their dw / db sums in registers; a workgroup adds up its row groups in LDS and writes one partial row, and a
// second launch adds the partial rows in a fixed order (no atomics: the same bits every time).
// 32768 x 4096 bf16 with a residual: forward 203 us (1.07 GB, 5.3 TB/s), backward 237 + 7 us (1.07 GB, 4.4 TB/s); a copy of
// 4 GiB reaches 4.8.  4096 x 1024 fp32: 8.8 and 12.8 + 4.0 us: there each of 1024 workgroups has one row group, so the partial
// rows (8.4 MB, 8 bytes for every element of up to 1024 row groups) are written for nothing that registers added up.
// Rows beyond the registers: 2000 x 20001 bf16 107 us forward (160 MB, 1.5 TB/s), 210 + 43 backward (element by element).
#include "lowp.h"
#include "../../include/rs_hip.h"

#pragma clang fp contract(fast)

namespace {

constexpr int EPT = 16;          // elements of a row per lane

// Sum over the LPR lanes of a row; every lane gets it.  LPR <= 64: within the wave.  Else over the workgroup, through a
// slot of `red` per wave; consecutive calls must use different slots (the caller alternates) so that one barrier does.
template <int LPR> __device__ __forceinline__ float row_sum(float v, float* red) {
    constexpr int W = LPR < 64 ? LPR : 64;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if constexpr (LPR > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < LPR / 64; ++i) v += red[i];
    }
    return v;
}
template <int LPR> __device__ __forceinline__ float2 row_sum2(float a, float b, float* red) {
    constexpr int W = LPR < 64 ? LPR : 64;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) { a += __shfl_xor(a, o, 64); b += __shfl_xor(b, o, 64); }
    if constexpr (LPR > 64) {
        if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = a; red[LPR / 64 + (threadIdx.x >> 6)] = b; }
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < LPR / 64; ++i) { a += red[i]; b += red[LPR / 64 + i]; }
    }
    return make_float2(a, b);
}

// E weights (or biases) from column n on: their type is T or fp32; absent ones are `other`.
template <typename T, bool WHOLE> __device__ __forceinline__ void load_param(const void* p, int is_f32, int n, int left, float other, float* v) {
    constexpr int E = RsVec<T>::E;
    if (!p) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = other;
    } else if (is_f32) {
#pragma unroll
        for (int q = 0; q < E; q += 4) rs_load<float, WHOLE>((const float*)p + n + q, left - q, v + q);
    } else {
        rs_load<T, WHOLE>((const T*)p + n, left, v);
    }
}
template <typename T> __device__ __forceinline__ float one_param(const void* p, int is_f32, int n, float other) {
    return !p ? other : is_f32 ? ((const float*)p)[n] : (float)((const T*)p)[n];
}

template <typename T, bool WHOLE, int LPR>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void layer_norm_fwd_kernel(
    const T* __restrict__ x, long long ldx, const T* __restrict__ r, long long ldr, int M, int N, const void* __restrict__ w,
    const void* __restrict__ b, int param_f32, float eps, T* __restrict__ y, T* __restrict__ s_out,
    float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    constexpr int NT = LPR > 256 ? LPR : 256, VE = RsVec<T>::E, CH = EPT / VE;
    __shared__ float red[2][NT / 64];
    const int t = threadIdx.x % LPR;
    const long long m = rs_block_id() * (NT / LPR) + threadIdx.x / LPR;
    const bool live = m < M;             // a row group past the last row goes along with the barriers and writes nothing
    float v[EPT];
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int n = (c * LPR + t) * VE;
        float* vc = v + c * VE;
        if (live && n < N) {
            rs_load<T, WHOLE>(x + m * ldx + n, N - n, vc);
            if (r) {
                float q[VE];
                rs_load<T, WHOLE>(r + m * ldr + n, N - n, q);
#pragma unroll
                for (int e = 0; e < VE; ++e) vc[e] = (float)(T)(vc[e] + q[e]);      // s is what its type holds
                rs_store<T, WHOLE>(s_out + m * N + n, N - n, vc);
            }
#pragma unroll
            for (int e = 0; e < VE; ++e) sum += vc[e];
        }
    }
    const float mu = row_sum<LPR>(sum, red[0]) / (float)N;
    float sq = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
        if ((c * LPR + t) * VE < N)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float d = v[c * VE + e] - mu;
                if (WHOLE || (c * LPR + t) * VE + e < N) sq += d * d;
            }
    const float rstd = 1.f / sqrtf(row_sum<LPR>(sq, red[1]) / (float)N + eps);
    if (!live) return;
    if (t == 0) {
        if (mean_out) mean_out[m] = mu;
        if (rstd_out) rstd_out[m] = rstd;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int n = (c * LPR + t) * VE;
        if (n < N) {
            float wv[VE], bv[VE], o[VE];
            load_param<T, WHOLE>(w, param_f32, n, N - n, 1.f, wv);
            load_param<T, WHOLE>(b, param_f32, n, N - n, 0.f, bv);
#pragma unroll
            for (int e = 0; e < VE; ++e) o[e] = (v[c * VE + e] - mu) * rstd * wv[e] + bv[e];
            rs_store<T, WHOLE>(y + m * N + n, N - n, o);
        }
    }
}

// Rows of any length, one per workgroup of 1024: mean, variance and output each walk over the row.
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_fwd_long_kernel(
    const T* __restrict__ x, long long ldx, const T* __restrict__ r, long long ldr, int M, int N, const void* __restrict__ w,
    const void* __restrict__ b, int param_f32, float eps, T* __restrict__ y, T* s_out, float* __restrict__ mean_out,
    float* __restrict__ rstd_out) {
    __shared__ float red[2][16];
    const long long m = rs_block_id();
    if (m >= M) return;
    const T* row = r ? s_out + m * N : x + m * ldx;
    float sum = 0.f;
    for (int n = threadIdx.x; n < N; n += 1024) {
        float v = (float)x[m * ldx + n];
        if (r) {
            const T s = (T)(v + (float)r[m * ldr + n]);
            s_out[m * N + n] = s;            // read back below by the lane that wrote it
            v = (float)s;
        }
        sum += v;
    }
    const float mu = row_sum<1024>(sum, red[0]) / (float)N;
    float sq = 0.f;
    for (int n = threadIdx.x; n < N; n += 1024) {
        const float d = (float)row[n] - mu;
        sq += d * d;
    }
    const float rstd = 1.f / sqrtf(row_sum<1024>(sq, red[1]) / (float)N + eps);
    if (threadIdx.x == 0) {
        if (mean_out) mean_out[m] = mu;
        if (rstd_out) rstd_out[m] = rstd;
    }
    for (int n = threadIdx.x; n < N; n += 1024) {
        y[m * N + n] = (T)(((float)row[n] - mu) * rstd * one_param<T>(w, param_f32, n, 1.f) + one_param<T>(b, param_f32, n, 0.f));
    }
}

// part: [gridDim.x, 2, N], dw sums in front of db sums.
template <typename T, bool WHOLE, int LPR>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void layer_norm_bwd_kernel(
    const T* __restrict__ dy, long long lddy, const T* __restrict__ s, long long lds, const float* __restrict__ mean,
    const float* __restrict__ rstd, const void* __restrict__ w, int param_f32, const T* __restrict__ ds, long long ldds, int M,
    int N, T* __restrict__ dx, float* __restrict__ part) {
    constexpr int NT = LPR > 256 ? LPR : 256, VE = RsVec<T>::E, CH = EPT / VE, R = NT / LPR;
    __shared__ float red[2][2 * (NT / 64)];
    __shared__ float fold[R > 1 ? R * LPR : 1];
    const int t = threadIdx.x % LPR, g = threadIdx.x / LPR;
    float dw[EPT], db[EPT], wv[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) dw[i] = db[i] = wv[i] = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int n = (c * LPR + t) * VE;
        if (n < N) load_param<T, WHOLE>(w, param_f32, n, N - n, 1.f, wv + c * VE);
    }
    const float inv = 1.f / (float)N;
    int turn = 0;
    // the trip count is the workgroup's, so that all its lanes meet at the barriers
    for (long long m0 = (long long)blockIdx.x * R; m0 < M; m0 += (long long)gridDim.x * R, turn ^= 1) {
        const long long m = m0 + g;
        const bool live = m < M;
        float mu = 0.f, rs = 0.f, s1 = 0.f, s2 = 0.f;
        float xh[EPT], gy[EPT];
        if (live) { mu = mean[m]; rs = rstd[m]; }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int n = (c * LPR + t) * VE;
            float* xc = xh + c * VE;
            float* gc = gy + c * VE;
            if (live && n < N) {
                rs_load<T, WHOLE>(s + m * lds + n, N - n, xc);
                rs_load<T, WHOLE>(dy + m * lddy + n, N - n, gc);
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    xc[e] = (xc[e] - mu) * rs;
                    dw[c * VE + e] += gc[e] * xc[e];
                    db[c * VE + e] += gc[e];
                    gc[e] *= wv[c * VE + e];
                    s1 += gc[e];
                    s2 += gc[e] * xc[e];
                }
            }
        }
        const float2 sums = row_sum2<LPR>(s1, s2, red[turn]);
        const float c1 = sums.x * inv, c2 = sums.y * inv;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int n = (c * LPR + t) * VE;
            if (live && n < N) {
                float o[VE];
#pragma unroll
                for (int e = 0; e < VE; ++e) o[e] = rs * (gy[c * VE + e] - c1 - xh[c * VE + e] * c2);
                if (ds) {
                    float q[VE];
                    rs_load<T, WHOLE>(ds + m * ldds + n, N - n, q);
#pragma unroll
                    for (int e = 0; e < VE; ++e) o[e] += q[e];
                }
                rs_store<T, WHOLE>(dx + m * N + n, N - n, o);
            }
        }
    }
    if (!part) return;
    float* pw = part + (long long)blockIdx.x * 2 * N;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const int n = (c * LPR + t) * VE + e;
            float a = dw[c * VE + e], b = db[c * VE + e];
            if constexpr (R > 1) {           // the row groups of the workgroup, in their order
                __syncthreads();
                fold[threadIdx.x] = a;
                __syncthreads();
                if (g == 0) {
                    a = 0.f;
#pragma unroll 8
                    for (int i = 0; i < R; ++i) a += fold[i * LPR + t];
                }
                __syncthreads();
                fold[threadIdx.x] = b;
                __syncthreads();
                if (g == 0) {
                    b = 0.f;
#pragma unroll 8
                    for (int i = 0; i < R; ++i) b += fold[i * LPR + t];
                }
            }
            if (g == 0 && n < N) { pw[n] = a; pw[N + n] = b; }
        }
}

template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_bwd_long_kernel(
    const T* __restrict__ dy, long long lddy, const T* __restrict__ s, long long lds, const float* __restrict__ mean,
    const float* __restrict__ rstd, const void* __restrict__ w, int param_f32, const T* __restrict__ ds, long long ldds, int M,
    int N, T* __restrict__ dx, float* __restrict__ part) {
    __shared__ float red[2][32];
    const float inv = 1.f / (float)N;
    float* pw = part ? part + (long long)blockIdx.x * 2 * N : nullptr;
    int turn = 0;
    bool first = true;
    for (long long m = blockIdx.x; m < M; m += gridDim.x, turn ^= 1, first = false) {
        const float mu = mean[m], rs = rstd[m];
        float s1 = 0.f, s2 = 0.f;
        for (int n = threadIdx.x; n < N; n += 1024) {
            const float xh = ((float)s[m * lds + n] - mu) * rs, d = (float)dy[m * lddy + n];
            const float wv = one_param<T>(w, param_f32, n, 1.f);
            s1 += d * wv;
            s2 += d * wv * xh;
            if (pw) {                        // a column belongs to one lane: no other touches its sums
                pw[n] = (first ? 0.f : pw[n]) + d * xh;
                pw[N + n] = (first ? 0.f : pw[N + n]) + d;
            }
        }
        const float2 sums = row_sum2<1024>(s1, s2, red[turn]);
        const float c1 = sums.x * inv, c2 = sums.y * inv;
        for (int n = threadIdx.x; n < N; n += 1024) {
            const float xh = ((float)s[m * lds + n] - mu) * rs;
            float o = rs * ((float)dy[m * lddy + n] * one_param<T>(w, param_f32, n, 1.f) - c1 - xh * c2);
            if (ds) o += (float)ds[m * ldds + n];
            dx[m * N + n] = (T)o;
        }
    }
}

// dw / db [N] from the partial rows: a workgroup of 1024 adds 32 columns, 32 lanes to a column.
template <typename W>
__global__ __launch_bounds__(1024) void layer_norm_params_kernel(const float* __restrict__ part, int rows, int N,
                                                                 W* __restrict__ dw, W* __restrict__ db) {
    __shared__ float fold[32][33];
    const int c = threadIdx.x & 31, r = threadIdx.x >> 5;
    const long long n = rs_block_id() * 32 + c, width = 2LL * N;
    float a = 0.f;
    if (n < width) {
#pragma unroll 8
        for (int i = r; i < rows; i += 32) a += part[i * width + n];
    }
    fold[r][c] = a;
    __syncthreads();
    if (r == 0 && n < width) {
        a = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) a += fold[i][c];
        if (n < N) {
            if (dw) dw[n] = (W)a;
        } else if (db) {
            db[n - N] = (W)a;
        }
    }
}

// Lanes per row, 0: the long form.
inline int lanes_for(int N) {
    const int choices[] = {8, 32, 64, 256, 1024};
    for (int l : choices)
        if ((long long)l * EPT >= N) return l;
    return 0;
}

struct NormArgs {
    const void *x, *r, *w, *b, *ds;
    long long ldx, ldr, ldds;
    int M, N, param_f32;
    float eps;
    void *y, *s;
    float *mean, *rstd;
};

// Aligned 16-byte accesses need every row of every operand to start at a multiple of 16 bytes.
inline bool vec_ok(int dtype, int N, long long ld, const void* p) {
    const int e = 16 / rs_elem_bytes(dtype);
    return !p || (rs_aligned16(p) && ld % e == 0 && N % e == 0);
}

template <typename T, bool WHOLE> int launch_fwd(const NormArgs& a, hipStream_t stream) {
    const int l = lanes_for(a.N);
    const T *x = (const T*)a.x, *r = (const T*)a.r;
#define RS_LN_FWD(L)                                                                                                          \
    case L:                                                                                                                   \
        hipLaunchKernelGGL((layer_norm_fwd_kernel<T, WHOLE, L>), rs_grid(rs_cdiv(a.M, (L > 256 ? L : 256) / L)),                 \
                           dim3(L > 256 ? L : 256), 0, stream, x, a.ldx, r, a.ldr, a.M, a.N, a.w, a.b, a.param_f32, a.eps,    \
                           (T*)a.y, (T*)a.s, a.mean, a.rstd);                                                                 \
        break;
    switch (l) {
        RS_LN_FWD(8)
        RS_LN_FWD(32)
        RS_LN_FWD(64)
        RS_LN_FWD(256)
        RS_LN_FWD(1024)
        default:
            hipLaunchKernelGGL((layer_norm_fwd_long_kernel<T>), rs_grid(a.M), dim3(1024), 0, stream, x, a.ldx, r, a.ldr, a.M, a.N,
                               a.w, a.b, a.param_f32, a.eps, (T*)a.y, (T*)a.s, a.mean, a.rstd);
    }
#undef RS_LN_FWD
    RS_CHECK_LAUNCH("rs_layer_norm_fwd");
    return RS_OK;
}

// y = dy, s, ds as inputs; b unused
template <typename T, bool WHOLE> int launch_bwd(const NormArgs& a, const void* dy, long long lddy, void* dx, float* part, int rows,
                                             hipStream_t stream) {
    const int l = lanes_for(a.N);
    const T *s = (const T*)a.x, *d = (const T*)dy, *ds = (const T*)a.ds;
#define RS_LN_BWD(L)                                                                                                          \
    case L:                                                                                                                   \
        hipLaunchKernelGGL((layer_norm_bwd_kernel<T, WHOLE, L>), dim3(rows), dim3(L > 256 ? L : 256), 0, stream, d, lddy, s,      \
                           a.ldx, a.mean, a.rstd, a.w, a.param_f32, ds, a.ldds, a.M, a.N, (T*)dx, part);                      \
        break;
    switch (l) {
        RS_LN_BWD(8)
        RS_LN_BWD(32)
        RS_LN_BWD(64)
        RS_LN_BWD(256)
        RS_LN_BWD(1024)
        default:
            hipLaunchKernelGGL((layer_norm_bwd_long_kernel<T>), dim3(rows), dim3(1024), 0, stream, d, lddy, s, a.ldx, a.mean,
                               a.rstd, a.w, a.param_f32, ds, a.ldds, a.M, a.N, (T*)dx, part);
    }
#undef RS_LN_BWD
    RS_CHECK_LAUNCH("rs_layer_norm_bwd");
    return RS_OK;
}

inline bool type_ok(int dtype, int param_dtype) {
    return (dtype == RS_F32 || dtype == RS_BF16 || dtype == RS_F16) && (param_dtype == dtype || param_dtype == RS_F32);
}

}  // namespace

extern "C" {

int rs_layer_norm_partial_rows(int M, int N) {
    if (M <= 0 || N <= 0) return 0;
    const int l = lanes_for(N), r = l && l < 256 ? 256 / l : 1;
    const int most = 1024;
    const int groups = rs_cdiv(M, r);
    return groups < most ? groups : most;
}

size_t rs_layer_norm_bwd_workspace_floats(int M, int N) { return (size_t)rs_layer_norm_partial_rows(M, N) * 2 * (N > 0 ? N : 0); }

int rs_layer_norm_fwd(int dtype, int param_dtype, const void* x, long long ldx, const void* r, long long ldr, int M, int N,
                      const void* w, const void* b, float eps, void* y, void* s, float* mean, float* rstd,
                      rs_stream_t stream) {
    RS_CHECK_ARG(type_ok(dtype, param_dtype), "rs_layer_norm_fwd: types %d / %d not served", dtype, param_dtype);
    RS_CHECK_ARG(M >= 0 && N > 0, "rs_layer_norm_fwd: bad shape %d x %d", M, N);
    if (M == 0) return RS_OK;
    RS_CHECK_ARG(x && y && (!r || s), "rs_layer_norm_fwd: null argument");
    RS_CHECK_ARG((M == 1 || ldx >= N) && (!r || M == 1 || ldr >= N), "rs_layer_norm_fwd: row strides are smaller than N");
    const NormArgs a = {x, r, w, b, nullptr, ldx, ldr, 0, M, N, param_dtype == RS_F32, eps, y, s, mean, rstd};
    const bool vec = vec_ok(dtype, N, M > 1 ? ldx : 0, x) && vec_ok(dtype, N, M > 1 ? ldr : 0, r) && rs_aligned16(y) &&
                     (!r || rs_aligned16(s)) && rs_aligned16(w) && rs_aligned16(b);
    if (dtype == RS_F32) return vec ? launch_fwd<float, true>(a, stream) : launch_fwd<float, false>(a, stream);
    if (dtype == RS_BF16) return vec ? launch_fwd<__bf16, true>(a, stream) : launch_fwd<__bf16, false>(a, stream);
    return vec ? launch_fwd<_Float16, true>(a, stream) : launch_fwd<_Float16, false>(a, stream);
}

int rs_layer_norm_bwd(int dtype, int param_dtype, const void* dy, long long lddy, const void* s, long long lds,
                      const float* mean, const float* rstd, const void* w, const void* ds, long long ldds, int M, int N,
                      void* dx, void* dw, void* db, float* workspace, size_t workspace_floats, rs_stream_t stream) {
    RS_CHECK_ARG(type_ok(dtype, param_dtype), "rs_layer_norm_bwd: types %d / %d not served", dtype, param_dtype);
    RS_CHECK_ARG(M >= 0 && N > 0, "rs_layer_norm_bwd: bad shape %d x %d", M, N);
    const bool params = dw || db;
    const int rows = rs_layer_norm_partial_rows(M, N);
    if (M > 0) {
        RS_CHECK_ARG(dy && s && mean && rstd && dx, "rs_layer_norm_bwd: null argument");
        RS_CHECK_ARG(M == 1 || (lddy >= N && lds >= N && (!ds || ldds >= N)),
                     "rs_layer_norm_bwd: row strides are smaller than N");
        if (params && (!workspace || workspace_floats < rs_layer_norm_bwd_workspace_floats(M, N))) {
            rs_set_error("rs_layer_norm_bwd: workspace of %zu floats, %zu needed", workspace_floats,
                         rs_layer_norm_bwd_workspace_floats(M, N));
            return RS_ERR_WORKSPACE;
        }
        const NormArgs a = {s, nullptr, w, nullptr, ds, lds, 0, ldds, M, N, param_dtype == RS_F32, 0.f, nullptr, nullptr,
                            (float*)mean, (float*)rstd};
        float* part = params ? workspace : nullptr;
        const bool vec = vec_ok(dtype, N, M > 1 ? lddy : 0, dy) && vec_ok(dtype, N, M > 1 ? lds : 0, s) &&
                         vec_ok(dtype, N, M > 1 ? ldds : 0, ds) && rs_aligned16(dx) && rs_aligned16(w);
        int rc;
        if (dtype == RS_F32)
            rc = vec ? launch_bwd<float, true>(a, dy, lddy, dx, part, rows, stream)
                     : launch_bwd<float, false>(a, dy, lddy, dx, part, rows, stream);
        else if (dtype == RS_BF16)
            rc = vec ? launch_bwd<__bf16, true>(a, dy, lddy, dx, part, rows, stream)
                     : launch_bwd<__bf16, false>(a, dy, lddy, dx, part, rows, stream);
        else
            rc = vec ? launch_bwd<_Float16, true>(a, dy, lddy, dx, part, rows, stream)
                     : launch_bwd<_Float16, false>(a, dy, lddy, dx, part, rows, stream);
        if (rc != RS_OK) return rc;
    }
    if (params) {                            // no rows: the sums are zero
        const dim3 grid = rs_grid((2LL * N + 31) / 32);
        if (param_dtype == RS_F32)
            hipLaunchKernelGGL(layer_norm_params_kernel<float>, grid, dim3(1024), 0, stream, workspace, rows, N, (float*)dw,
                               (float*)db);
        else if (param_dtype == RS_BF16)
            hipLaunchKernelGGL(layer_norm_params_kernel<__bf16>, grid, dim3(1024), 0, stream, workspace, rows, N, (__bf16*)dw,
                               (__bf16*)db);
        else
            hipLaunchKernelGGL(layer_norm_params_kernel<_Float16>, grid, dim3(1024), 0, stream, workspace, rows, N,
                               (_Float16*)dw, (_Float16*)db);
        RS_CHECK_LAUNCH("rs_layer_norm_bwd");
    }
    return RS_OK;
}

}  // extern "C"
