// Attention where a sample has few keys and rows -- the fields of a sample, short histories: at most 64 rows, and keys times
// head elements (in tiles of 16) up to 64 x 32 in fp32, 64 x 64 in 16 bits.  The formulas and masks are those of
// attention.hip.
//
// One wave per (sample, head), nothing shared with others: no barriers.  Keys and values (all of them) lie in the wave's
// LDS, padded so that consecutive rows start 4 banks (mod 64) apart; the query rows pass by in tiles of 16 and stay in
// registers.  16x16 matrix tiles: 39 fields fill 48 rows and columns, where 32x32 tiles would pad them to 64 by 64 and a
// head of 16 to 32.  As in attention.hip the scores of a column's row stay in its lanes and go into the next product as
// they are.
// The backward makes the scores once: dq comes from the columns as they are, and for dk and dv, whose contraction runs
// over the rows, P and dS of a row tile go through a small LDS tile to be read the other way.  The query heads that
// share a key head pass by one after the other, so every gradient has one owner.  A wave has a row's whole P and do . v, so
// delta_i = sum_j p_ij (do_i . v_j), which is the same as do_i . o_i without o and its rounding.
// 39 fields x 4096 samples, 2 heads of 16, fp32: forward 27 us (82 MB, 3.0 TB/s), backward 53 us (143 MB, 2.7 TB/s), of which
// 8 and 19 us are matrix instructions; what is left is the latency of each wave's one short chain.
#include "attention.h"

#pragma clang fp contract(fast)

namespace {

// What lanes wrote to LDS in front of it is what other lanes of the wave read behind it, and what was read in front of it may
// be written over.  The hardware runs a wave's LDS accesses in their order, so this costs no instruction; it holds the
// compiler to that order, which sees one lane's addresses only.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Rows of W elements in LDS, 16 bytes of padding to a row.
template <typename T, int W> struct Rows {
    static constexpr int E = Mma16<T>::E, RS = W + E;
    typedef typename Mma16<T>::V V;
    static __device__ __forceinline__ V rows(const T* lds, int row0, int c) {
        const int l = threadIdx.x & 63;
        return *(const V*)(lds + (row0 + (l & 15)) * RS + c * Mma16<T>::CK + (l >> 4) * E);
    }
    // transposed: element col0 + l % 16 of the rows a result's registers hold, from tile row0 on (TILES of them)
    static __device__ __forceinline__ V cols(const T* lds, int row0, int col0) {
        const int l = threadIdx.x & 63;
        if constexpr (sizeof(T) == 4) {
            V r;
            const T* p = lds + (row0 + 4 * (l >> 4)) * RS + col0 + (l & 15);
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = p[i * RS];
            return r;
        } else {
            const T* p = lds + (row0 + 4 * (l >> 4) + ((l & 15) >> 2)) * RS + col0 + 4 * (l & 3);
            typedef __attribute__((address_space(3))) rs_s16x4* lds_ptr;
            union { rs_s16x4 s[2]; V v; } f;
            f.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p);
            f.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 16 * RS));
            return f.v;
        }
    }
};

// R rows from row0 on to LDS: rows outside [begin, end) and columns from D on become zeros.
template <typename T, int W, int R, bool VEC> struct Copy {
    static constexpr int E = Mma16<T>::E, UPR = W / E, N = (R * UPR + 63) / 64;
    typename Mma16<T>::V r[N];
    __device__ __forceinline__ void load(const T* base, long long stride, int row0, int begin, int end, int D) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int x = (threadIdx.x & 63) + i * 64, row = row0 + x / UPR;
            r[i] = fetch<T, VEC>(base + row * stride, x % UPR * E, D, x < R * UPR && row >= begin && row < end);
        }
    }
    __device__ __forceinline__ void store(T* lds) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int x = (threadIdx.x & 63) + i * 64;
            if (x < R * UPR) *(typename Mma16<T>::V*)(lds + x / UPR * Rows<T, W>::RS + x % UPR * E) = r[i];
        }
    }
};

// B operand of a contraction over rows from the results of TILES row tiles.
template <typename T> __device__ __forceinline__ typename Mma16<T>::V pack(const rs_f32x4* s) {
    typename Mma16<T>::V r;
#pragma unroll
    for (int e = 0; e < Mma16<T>::E; ++e) r[e] = (T)s[e / 4][e % 4];
    return r;
}
// Keys [0, keys) and rows [begin, rows) that have a part in sample b (row_limit says which goes with which).
struct Part {
    int keys, begin, rows;
    long long start;
};
__device__ __forceinline__ Part part_of(const AttnArgs& a, int b) {
    Part p;
    p.rows = a.qlen ? min(max(a.qlen[b], 0), a.Tq) : a.Tq;
    p.keys = a.len ? min(max(a.len[b], 0), a.Tk) : a.Tk;
    p.start = a.qstart ? a.qstart[b] : a.start;
    p.begin = 0;
    if (a.causal) {
        p.begin = p.start < 0 ? (int)min(-p.start, (long long)p.rows) : 0;
        p.keys = (int)max(0LL, min((long long)p.keys, p.start + p.rows));
    }
    if (p.keys == 0) p.begin = p.rows;
    if (p.begin == p.rows) p.keys = 0;
    return p;
}
// What row i sees: keys below the result.
__device__ __forceinline__ int limit(const AttnArgs& a, const Part& p, int i) {
    if (i < p.begin || i >= p.rows) return 0;
    return a.causal ? (int)min((long long)p.keys, p.start + i + 1) : p.keys;
}

// Workgroup -> (sample, head), sample >= B: none.  Workgroups go round the eight XCDs; the heads of a sample, whose rows
// share cache lines (a head of 16 fp32 elements is half of one), go to one XCD where there are samples enough for all.
struct Unit {
    int b, h;
};
__device__ __forceinline__ Unit unit_of(const AttnArgs& a, int heads) {
    const unsigned id = (unsigned)rs_block_id(), n = heads;
    if (!a.dealt) return {(int)(id / n), (int)(id % n)};
    const unsigned j = id >> 3, k = j / n;
    return {(int)(k * 8 + (id & 7)), (int)(j - k * n)};
}

// ---- forward -----------------------------------------------------------------------------------------------------
// NT: tiles of 16 keys.  A workgroup is one wave with one head of one sample.
template <typename T, int DP, int NT, bool VEC>
__global__ __launch_bounds__(64) void attention_small_fwd_kernel(const AttnArgs a) {
    constexpr int CK = Mma16<T>::CK, E = Mma16<T>::E, TILES = Mma16<T>::TILES, NC = DP / CK, ND = DP / 16;
    typedef typename Mma16<T>::V V;
    typedef Rows<T, DP> L;
    __shared__ __align__(16) T s_k[NT * 16 * L::RS];
    __shared__ __align__(16) T s_v[NT * 16 * L::RS];
    const int Hq = a.Hk * a.G;
    const Unit unit = unit_of(a, Hq);
    if (unit.b >= a.B) return;
    const int b = unit.b, h = unit.h, hk = (unsigned)h / (unsigned)a.G;
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const Part part = part_of(a, b);
    const float scale2 = a.scale * LOG2E;
    const T* q = row_ptr<T>(a.q, b, 0, h);
    Copy<T, DP, NT * 16, VEC> ck, cv;
    ck.load(row_ptr<T>(a.k, b, 0, hk), a.k.t, 0, 0, part.keys, a.D);
    cv.load(row_ptr<T>(a.v, b, 0, hk), a.v.t, 0, 0, part.keys, a.D);
    V qf[NC], qn[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) qn[c] = fetch<T, VEC>(q + (long long)col * a.q.t, c * CK + g * E, a.D, col >= part.begin && col < part.rows);
    ck.store(s_k);
    cv.store(s_v);
    wave_sync();
    for (int i0 = 0; i0 < a.Tq; i0 += 16) {
        const int i = i0 + col, lim = limit(a, part, i);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            qf[c] = qn[c];
            const int next = i + 16;
            qn[c] = fetch<T, VEC>(q + (long long)next * a.q.t, c * CK + g * E, a.D, next >= part.begin && next < part.rows);
        }
        rs_f32x4 s[NT];
        float m = -INFINITY;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            s[n] = rs_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NC; ++c) s[n] = Mma16<T>::mul(L::rows(s_k, n * 16, c), qf[c], s[n]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (n * 16 + 4 * g + e >= lim) s[n][e] = -INFINITY;
                m = fmaxf(m, s[n][e]);
            }
        }
        m = col_max(m) * scale2;
        const float base = m == -INFINITY ? 0.f : m;
        float l = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[n][e] = __builtin_amdgcn_exp2f(s[n][e] * scale2 - (base - P_SHIFT<T>));
                l += s[n][e];
            }
        l = col_sum(l);
        rs_f32x4 o[ND];
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = rs_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NT; n += TILES) {
            const V p = pack<T>(s + n);
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] = Mma16<T>::mul(L::cols(s_v, n * 16, d * 16), p, o[d]);
        }
        if (i >= a.Tq) continue;
        const bool none = l == 0.f;                               // nothing seen: zeros, whatever the other rows' keys hold
        const float inv = 1.f / l;
        if (a.lse && g == 0) a.lse[((long long)b * Hq + h) * a.Tq + i] = none ? -INFINITY : (m + log2f(l) - P_SHIFT<T>) * LN2;
        T* out = (T*)a.out + (((long long)b * a.Tq + i) * Hq + h) * a.D;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = none ? 0.f : o[d][e] * inv;
            store4<T>(out, d * 16 + 4 * g, a.D, a.out_vec, x);
        }
    }
}

// ---- backward ------------------------------------------------------------------------------------------------------
// A wave per (sample, key head).  Row tiles go TILES at a time, what one contraction step over rows takes.
template <typename T, int DP, int NT, bool VEC>
__global__ __launch_bounds__(64) void attention_small_bwd_kernel(const AttnArgs a) {
    constexpr int CK = Mma16<T>::CK, TILES = Mma16<T>::TILES, NC = DP / CK, ND = DP / 16, R = 16 * TILES;
    constexpr bool F16 = P_SHIFT<T> != 0.f;
    typedef typename Mma16<T>::V V;
    typedef Rows<T, DP> L;
    typedef Rows<T, NT * 16> LP;
    __shared__ __align__(16) T s_k[NT * 16 * L::RS];
    __shared__ __align__(16) T s_v[NT * 16 * L::RS];
    __shared__ __align__(16) T s_q[R * L::RS];
    __shared__ __align__(16) T s_g[R * L::RS];
    __shared__ __align__(16) T s_p[R * LP::RS];
    __shared__ __align__(16) T s_d[R * LP::RS];
    const Unit unit = unit_of(a, a.Hk);
    if (unit.b >= a.B) return;
    const int b = unit.b, hk = unit.h, Hq = a.Hk * a.G;
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const Part part = part_of(a, b);
    const float scale2 = a.scale * LOG2E;
    Copy<T, DP, NT * 16, VEC> ck, cv;
    Copy<T, DP, R, VEC> cq, cg;
    ck.load(row_ptr<T>(a.k, b, 0, hk), a.k.t, 0, 0, part.keys, a.D);
    cv.load(row_ptr<T>(a.v, b, 0, hk), a.v.t, 0, 0, part.keys, a.D);
    rs_f32x4 dk[NT][ND], dv[NT][ND];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int d = 0; d < ND; ++d) dk[n][d] = dv[n][d] = rs_f32x4{0.f, 0.f, 0.f, 0.f};
    Range range;                                                  // of all rows and keys: dS of a turn goes into one product
    // a turn is R rows of one head; loads run one turn ahead, as does the lanes' lse
    float lse[TILES];
    const int per_head = (a.Tq + R - 1) / R, turns = per_head * a.G;
    auto load = [&](int turn) {
        const int h = hk * a.G + turn / per_head, i0 = turn % per_head * R;
        cq.load(row_ptr<T>(a.q, b, 0, h), a.q.t, i0, part.begin, part.rows, a.D);
        cg.load(row_ptr<T>(a.go, b, 0, h), a.go.t, i0, part.begin, part.rows, a.D);
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int i = i0 + t * 16 + col;
            lse[t] = i >= part.begin && i < part.rows ? a.lse[((long long)b * Hq + h) * a.Tq + i] : INFINITY;
        }
    };
    if (turns > 0) load(0);
    ck.store(s_k);
    cv.store(s_v);
    for (int turn = 0; turn < turns; ++turn) {
        const int h = hk * a.G + turn / per_head, i0 = turn % per_head * R;
        wave_sync();                                              // the last turn's reads are done
        cq.store(s_q);
        cg.store(s_g);
        wave_sync();
        float lse2[TILES];
#pragma unroll
        for (int t = 0; t < TILES; ++t) lse2[t] = back_lse(lse[t]) - P_SHIFT<T>;
        if (turn + 1 < turns) load(turn + 1);
        rs_f32x4 all[TILES][NT];
        float most = 0.f;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int i = i0 + t * 16 + col, lim = limit(a, part, i);
            rs_f32x4 p[NT], (&ds)[NT] = all[t];
            float delta = 0.f, top = 0.f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                p[n] = ds[n] = rs_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    p[n] = Mma16<T>::mul(L::rows(s_k, n * 16, c), L::rows(s_q, t * 16, c), p[n]);
                    ds[n] = Mma16<T>::mul(L::rows(s_v, n * 16, c), L::rows(s_g, t * 16, c), ds[n]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool seen = n * 16 + 4 * g + e < lim;       // selected, not multiplied
                    p[n][e] = seen ? __builtin_amdgcn_exp2f(p[n][e] * scale2 - lse2[t]) : 0.f;
                    ds[n][e] = seen ? ds[n][e] : 0.f;
                    delta += p[n][e] * ds[n][e];
                }
            }
            delta = col_sum(delta) * P_UNIT<T>;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    ds[n][e] = p[n][e] * (ds[n][e] - delta);
                    top = fmaxf(top, fabsf(ds[n][e]));
                }
                // row = query: four consecutive keys of one row
                store4<T>(s_p + (t * 16 + col) * LP::RS, n * 16 + 4 * g, NT * 16, true, (const float*)&p[n]);
                if constexpr (!F16) store4<T>(s_d + (t * 16 + col) * LP::RS, n * 16 + 4 * g, NT * 16, true, (const float*)&ds[n]);
            }
            float back = a.scale;                                 // dq takes a factor for each row
            rs_f32x4 own[NT];
            if constexpr (F16) {
                top = col_max(top);
                most = fmaxf(most, top);
                Range row;
                const int by = row.follow(top);
                back *= P_UNIT<T> * row.unit();
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) own[n][e] = ldexpf(ds[n][e], by);
            }
            rs_f32x4 dq[ND];
#pragma unroll
            for (int d = 0; d < ND; ++d) dq[d] = rs_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int n = 0; n < NT; n += TILES) {
                const V x = pack<T>((F16 ? own : ds) + n);
#pragma unroll
                for (int d = 0; d < ND; ++d) dq[d] = Mma16<T>::mul(L::cols(s_k, n * 16, d * 16), x, dq[d]);
            }
            if (i < a.Tq) {
                T* out = (T*)a.dq + (((long long)b * a.Tq + i) * Hq + h) * a.D;
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = lim == 0 || lse2[t] == INFINITY ? 0.f : dq[d][e] * back;      // saw nothing
                    store4<T>(out, d * 16 + 4 * g, a.D, a.out_vec, x);
                }
            }
        }
        if constexpr (F16) {
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
            const int by = range.follow(ldexpf(most, range.exp));
            if (by != 0)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int e = 0; e < 4; ++e) dk[n][d][e] = ldexpf(dk[n][d][e], by);
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = ldexpf(all[t][n][e], range.exp);
                    store4<T>(s_d + (t * 16 + col) * LP::RS, n * 16 + 4 * g, NT * 16, true, x);
                }
        }
        wave_sync();
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const V p = LP::cols(s_p, 0, n * 16), ds = LP::cols(s_d, 0, n * 16);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                dv[n][d] = Mma16<T>::mul(L::cols(s_g, 0, d * 16), p, dv[n][d]);
                dk[n][d] = Mma16<T>::mul(L::cols(s_q, 0, d * 16), ds, dk[n][d]);
            }
        }
    }
    const float back = a.scale * P_UNIT<T> * range.unit();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int key = n * 16 + col;
        if (key >= a.Tk) continue;
        const long long at = (((long long)b * a.Tk + key) * a.Hk + hk) * a.D;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const float x[4] = {dk[n][d][0] * back, dk[n][d][1] * back, dk[n][d][2] * back, dk[n][d][3] * back};
            const float y[4] = {dv[n][d][0] * P_UNIT<T>, dv[n][d][1] * P_UNIT<T>, dv[n][d][2] * P_UNIT<T>, dv[n][d][3] * P_UNIT<T>};
            store4<T>((T*)a.dk + at, d * 16 + 4 * g, a.D, a.out_vec, x);
            store4<T>((T*)a.dv + at, d * 16 + 4 * g, a.D, a.out_vec, y);
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------
template <typename T, int DP, int NT> int launch(AttnArgs a, bool back, hipStream_t stream) {
    a.dealt = a.B >= 64;
    const dim3 grid = rs_grid((a.dealt ? (a.B + 7LL) / 8 * 8 : a.B) * a.Hk * (back ? 1 : a.G));
    if (back && a.vec) hipLaunchKernelGGL((attention_small_bwd_kernel<T, DP, NT, true>), grid, dim3(64), 0, stream, a);
    else if (back) hipLaunchKernelGGL((attention_small_bwd_kernel<T, DP, NT, false>), grid, dim3(64), 0, stream, a);
    else if (a.vec) hipLaunchKernelGGL((attention_small_fwd_kernel<T, DP, NT, true>), grid, dim3(64), 0, stream, a);
    else hipLaunchKernelGGL((attention_small_fwd_kernel<T, DP, NT, false>), grid, dim3(64), 0, stream, a);
    RS_CHECK_LAUNCH(back ? "rs_attention_bwd" : "rs_attention_fwd");
    return RS_OK;
}
// The kernel of the smallest head and tile count that cover D and Tk; together they cover what small_ok admits.
int launch_f32(const AttnArgs& a, bool back, hipStream_t stream) {
    const int n = a.Tk <= 16 ? 1 : (a.Tk + 15) / 16;
#define RS_SMALL(DP, NT) \
    if (a.D <= DP && n <= NT) return launch<float, DP, NT>(a, back, stream)
    RS_SMALL(16, 1);
    RS_SMALL(16, 2);
    RS_SMALL(16, 3);
    RS_SMALL(16, 4);
    RS_SMALL(32, 1);
    RS_SMALL(32, 2);
    RS_SMALL(32, 3);
    RS_SMALL(32, 4);
    RS_SMALL(64, 1);
    RS_SMALL(64, 2);
    RS_SMALL(128, 1);
    rs_set_error("attention: %d keys of %d elements are no small shape", a.Tk, a.D);
    return RS_ERR_ARG;
}
template <typename T> int launch_16(const AttnArgs& a, bool back, hipStream_t stream) {
    const int n = (a.Tk + 15) / 16;
#define RS_SMALL16(DP, NT) \
    if (a.D <= DP && n <= NT) return launch<T, DP, NT>(a, back, stream)
    RS_SMALL16(32, 2);
    RS_SMALL16(32, 4);
    RS_SMALL16(64, 2);
    RS_SMALL16(64, 4);
    RS_SMALL16(128, 2);
    rs_set_error("attention: %d keys of %d elements are no small shape", a.Tk, a.D);
    return RS_ERR_ARG;
}
int launch_any(int dtype, const AttnArgs& a, bool back, hipStream_t stream) {
    if (dtype == RS_F32) return launch_f32(a, back, stream);
    return dtype == RS_BF16 ? launch_16<__bf16>(a, back, stream) : launch_16<_Float16>(a, back, stream);
}

}  // namespace

// Against the kernels of attention.hip, forward and backward: 512 x 60 x 8 heads of 64 bf16 29 + 71 us (30 + 90), 1024 x 30 x 8
// of 128 bf16 61 + 120 (63 + 259), of 64 fp32 62 + 122 (71 + 469), 1024 x 16 x 8 of 128 fp32 60 + 104 (172 + 517).  Larger
// products than these do not fit a wave's registers.
bool rs_attention_small_ok(int dtype, int Tq, int Tk, int D) {
    const int most = dtype == RS_F32 ? (D <= 32 ? 64 : D <= 64 ? 32 : 16) : (D <= 64 ? 64 : 32);
    return Tq <= 64 && Tk <= most && D <= 128;
}
int rs_attention_small_fwd(int dtype, const AttnArgs& a, hipStream_t stream) { return launch_any(dtype, a, false, stream); }
int rs_attention_small_bwd(int dtype, const AttnArgs& a, hipStream_t stream) { return launch_any(dtype, a, true, stream); }
