// Attention over fields, histories and cached keys: forward, backward and single tokens; fp32, bf16 and fp16, heads of up
// to 128 elements, several query heads to a key head.
//
//   z_ij = scale q_i . k_j,  p_ij = exp(z_ij - lse_i) over the keys row i sees,  o_i = sum_j p_ij v_j
//   delta_i = sum_d do_id o_id,  ds_ij = p_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
// Row i of sample b sees key j where j < lengths[b], i < query_lengths[b] and, causal, j <= i + query_start[b].  A row that
// sees nothing has o = 0, lse = -inf and no part in any gradient; what lies in keys and rows behind the lengths is never
// multiplied with anything.
//
// One pass over the keys with the running maximum and sum of the softmax; no matrix of scores exists.  All products run on
// the matrix cores as 32x32 tiles, always "A from LDS, B from registers": the fixed operand of a wave (its 32 query
// rows, or its 32 keys) stays in registers as columns, tiles of the other one pass through LDS.  The result of such a
// product holds one column per lane (and its partner lane + 32), 16 rows each, which is the layout the next product
// wants as its B operand if the contraction runs over the rows in the order the registers hold them: the scores turn into
// probabilities and go into the next product without leaving their lane.  The transposed A operands of that product
// (v, k, q, do with the head dimension as rows) are read from the same LDS tile, 16-bit types with the transposing LDS load.
//   forward   S^T = K Q^T, softmax down the lane's own registers, O^T += V^T P^T
//   dq        S^T, dP^T = V dO^T, dQ^T += K^T dS^T;  delta is made here and left for the other one
//   dk, dv    S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS
// The backward makes the scores twice (14 D instead of 10 D operations per pair) so that every gradient has one owner: no
// atomics, the same bits every time.  Query heads that share a key head lie next to one another as rows of the forward
// and dq (row = position * group + head), so a cache is read once for all of them; dk / dv walk over them.
//
// Bound by the matrix cores for heads of 128 (2 x 8192 x 16 heads on 4 key heads, bf16, causal: forward 551 us = 1000 TFLOP/s,
// dq 721 = 1140, dk / dv 1120 + 25 for the join = 960; a library product of 8192^3 reaches 1208 here), by the exponentials
// and the latency of a wave's chain for smaller ones (1537 x 12 x 3 heads of 64, fp16: 41 us, 530 TFLOP/s), by memory for
// single tokens over caches (1.07 GB of full caches in 190 us, 5.6 TB/s).  Heads between the padded sizes of 32, 64 and 128 pay
// for the padding: heads of 96 in the shape above 521, 667 and 1086 + 19 us.
//
// Roundings: products of 16-bit operands are exact and summed in fp32; P and dS are rounded to the operands' type for
// their second product (the matrix cores take equal types; the rounding is a half step per element and averages out over
// the keys).  With delta from the rounded o, dS would leave dq and dk of short rows 1.6 times as far off as their own last
// rounding; for heads up to 64, where the matrix cores have time, it is multiplied in two parts, its rounding and the rest
// of it (256 histories of 0..200, 8 heads of 32: 1.54 -> 1.03 times, for dq 39 -> 44 us and dk / dv 52 -> 57).  In fp16 P and dS
// are rounded as multiples of powers of two that keep them in the type's range (attention.h).  All statistics, sums and outputs before their last rounding are fp32.
#include "attention.h"
#include "../../include/rs_hip.h"

#pragma clang fp contract(fast)

namespace {

// Matrix tiles of one element type.  CK: elements of the contraction in one fragment pair; a fragment is 16 bytes a lane.
template <typename T> struct Mma;
template <> struct Mma<float> {
    static constexpr int CK = 8, E = 4;
    static constexpr bool F16 = false;
    typedef rs_f32x4 V;
    static __device__ __forceinline__ rs_f32x16 mul(V a, V b, rs_f32x16 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};
template <> struct Mma<__bf16> {
    static constexpr int CK = 16, E = 8;
    static constexpr bool F16 = false;
    typedef rs_bf16x8 V;
    static __device__ __forceinline__ rs_f32x16 mul(V a, V b, rs_f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct Mma<_Float16> {
    static constexpr int CK = 16, E = 8;
    static constexpr bool F16 = true;
    typedef rs_f16x8 V;
    static __device__ __forceinline__ rs_f32x16 mul(V a, V b, rs_f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

// A tile of rows in LDS, DP elements to a row in units of 16 bytes, unit u of row r in place u ^ swz(r): 16 rows at one unit
// (the direct fragment) and 8 rows by four neighbouring units (the transposed one) both spread over all 64 banks, and a
// row keeps its place in memory order, which is what the loads into LDS need.
template <typename T, int DP> struct Tile {
    static constexpr int E = Mma<T>::E, UPR = DP / E;
    typedef typename Mma<T>::V V;
    static __device__ __forceinline__ int swz(int r) {
        if constexpr (UPR >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
        else if constexpr (UPR == 8) return ((r & 2) << 1) | ((r >> 2) & 3);
        else return (r >> 2) & 3;
    }
    // rows row0 + lane % 32 (row0 a multiple of 32), elements of contraction step c
    static __device__ __forceinline__ V rows(const T* lds, int row0, int c) {
        const int l = threadIdx.x & 63, r = l & 31;
        return *(const V*)(lds + (row0 + r) * DP + (((2 * c + (l >> 5)) ^ swz(r)) * E));
    }
    // transposed: element col0 + lane % 32 of the rows that the registers of a product hold for contraction step c --
    // half h of the wave has rows 4h .. 4h+3 of each group of eight; row0 is a multiple of CK
    static __device__ __forceinline__ V cols(const T* lds, int row0, int col0) {
        const int l = threadIdx.x & 63;
        if constexpr (sizeof(T) == 4) {
            V v;
            const int col = col0 + (l & 31);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = row0 + 4 * (l >> 5) + i;
                v[i] = lds[r * DP + ((col / E) ^ swz(r)) * E + col % E];
            }
            return v;
        } else {
            // 16 lanes read 4 rows of 16 elements and get one element of each row
            const int r = row0 + 4 * (l >> 5) + ((l & 15) >> 2), col = col0 + 16 * ((l >> 4) & 1) + 4 * (l & 3);
            typedef __attribute__((address_space(3))) rs_s16x4* lds_ptr;
            union { rs_s16x4 s[2]; V v; } f;
            f.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds + r * DP + ((col / E) ^ swz(r)) * E + col % E));
            f.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds + (r + 8) * DP + ((col / E) ^ swz(r + 8)) * E + col % E));
            return f.v;
        }
    }
};

// G asynchronous 16-byte loads a lane, the first one's to LDS byte address dst, each further one's STEP behind.  m0, which
// takes the address, is the compiler's and cannot be declared overwritten: every statement gives it back.  The nops: m0 and
// descriptor registers that were written just before, the latter by vector instructions.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
template <int G, int STEP> __device__ __forceinline__ void loads_to_lds(unsigned dst, u32x4 rsrc, const unsigned* off) {
    static_assert(G == 1 || G == 2 || G == 4, "as many as the statements have");
    unsigned m0;
    if constexpr (G == 1)
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %3, %2, 0 offen lds\n\t"
                     "s_mov_b32 m0, %0"
                     : "=&s"(m0) : "s"(dst), "s"(rsrc), "v"(off[0]) : "memory");
    else if constexpr (G == 2)
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %4, %2, 0 offen lds\n\t"
                     "s_add_u32 m0, m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %5, %2, 0 offen lds\n\t"
                     "s_mov_b32 m0, %0"
                     : "=&s"(m0) : "s"(dst), "s"(rsrc), "i"(STEP), "v"(off[0]), "v"(off[1]) : "memory", "scc");
    else
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %4, %2, 0 offen lds\n\t"
                     "s_add_u32 m0, m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %5, %2, 0 offen lds\n\t"
                     "s_add_u32 m0, m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %6, %2, 0 offen lds\n\t"
                     "s_add_u32 m0, m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %7, %2, 0 offen lds\n\t"
                     "s_mov_b32 m0, %0"
                     : "=&s"(m0) : "s"(dst), "s"(rsrc), "i"(STEP), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]) : "memory", "scc");
}

// The way of consecutive tiles of R rows into LDS, NT lanes; rows from row_end on and columns from D on become zeros.
// VEC: asynchronous 16-byte loads from memory to LDS through a buffer descriptor that ends with the last row, whose range
// check supplies the zeros; no register holds the data, and the tile is there after the wait in feed_sync().
// Else (rows that do not start at multiples of 16 bytes): element by element through registers, land() writes them to LDS.
template <typename T, int DP, int R, int NT, bool VEC> struct Feed {
    typedef Tile<T, DP> L;
    typedef typename Mma<T>::V V;
    static constexpr int E = Mma<T>::E, UPR = L::UPR, N = R * UPR / NT;
    static_assert(R * UPR % NT == 0, "the lanes share a tile evenly");
    unsigned off[VEC ? N : 1];
    V reg[VEC ? 1 : N];
    const T* at;                 // first row of the next tile
    long long stride, left;      // left: elements from there to the end of the last row
    int rows, D;

    __device__ __forceinline__ Feed(long long row_stride, int d) : stride(row_stride), D(d) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int x = threadIdx.x + i * NT, r = x / UPR, u = (x % UPR) ^ L::swz(r);
                off[i] = u * E < D ? (unsigned)(r * stride * sizeof(T) + u * 16) : 0x7ffffff0u;
            }
        }
    }
    // the next tile is row0's (the same in all lanes)
    __device__ __forceinline__ void seek(const T* base, int row0, int row_end) {
        at = base + row0 * stride;
        rows = row_end - row0;
        left = (rows - 1) * stride + D;
    }
    __device__ __forceinline__ void next(T* lds) {
        if constexpr (VEC) {
            const unsigned long long where = (unsigned long long)at;
            const long long most = 0x7fffff00LL / (int)sizeof(T);
            const int bytes = (int)(left < most ? left : most) * (int)sizeof(T);
            const u32x4 rsrc = {(unsigned)__builtin_amdgcn_readfirstlane((int)where),
                                (unsigned)__builtin_amdgcn_readfirstlane((int)(where >> 32)) & 0xffffu,
                                (unsigned)__builtin_amdgcn_readfirstlane(bytes), 0x00027000u};
            const unsigned dst = __builtin_amdgcn_readfirstlane(
                (int)(unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)lds + (int)(threadIdx.x >> 6) * 1024);
#pragma unroll
            for (int i = 0; i < N; i += N < 4 ? N : 4) loads_to_lds<N < 4 ? N : 4, NT * 16>(dst + i * NT * 16, rsrc, off + i);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int x = threadIdx.x + i * NT, r = x / UPR, u = (x % UPR) ^ L::swz(r);
                reg[i] = fetch<T, false>(at + r * stride, u * E, D, r < rows);
            }
        }
        at += R * stride;
        rows -= R;
        left -= R * stride;
    }
    __device__ __forceinline__ void land(T* lds) const {
        if constexpr (!VEC) {
#pragma unroll
            for (int i = 0; i < N; ++i) *(V*)(lds + (threadIdx.x + i * NT) * E) = reg[i];
        }
    }
};
// This wave's loads have arrived and its reads are done, then everybody's.
template <bool VEC> __device__ __forceinline__ void feed_sync() {
    if constexpr (VEC) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else __syncthreads();
}

// The registers of contraction step c of a product as the next product's B operand.
template <typename T> __device__ __forceinline__ typename Mma<T>::V pack(const rs_f32x16& s, int c) {
    typename Mma<T>::V r;
#pragma unroll
    for (int e = 0; e < Mma<T>::E; ++e) r[e] = (T)s[c * Mma<T>::E + e];
    return r;
}

// What pack() rounds away, in the same places.
template <typename T> __device__ __forceinline__ typename Mma<T>::V pack_rest(const rs_f32x16& s, int c, typename Mma<T>::V p) {
    typename Mma<T>::V r;
#pragma unroll
    for (int e = 0; e < Mma<T>::E; ++e) r[e] = (T)(s[c * Mma<T>::E + e] - (float)p[e]);
    return r;
}

// Over a lane and its partner lane + 32 (both get it): the swap leaves the lower half's values in .x, the upper one's in .y.
__device__ __forceinline__ float2 halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_max(float x) {
    const float2 h = halves(x);
    return fmaxf(h.x, h.y);
}
__device__ __forceinline__ float half_sum(float x) {
    const float2 h = halves(x);
    return h.x + h.y;
}
__device__ __forceinline__ float reg_max(const rs_f32x16& s) {      // of the absolute values, NaN ignored
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) m = fmaxf(m, fabsf(s[e]));
    return m;
}
__device__ __forceinline__ void scale_by(rs_f32x16& s, int exp) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = ldexpf(s[e], exp);
}
// Row of register i within a 32x32 result.
__device__ __forceinline__ int reg_row(int i) { return 8 * (i >> 2) + 4 * ((threadIdx.x & 63) >> 5) + (i & 3); }

// Workgroup -> (sample, key head) pair, tile and share; pair < 0: no work.  Workgroups go round the eight XCDs: all work on
// one pair, which reads the same keys, gets to one XCD and its L2.  Many pairs are dealt out, up to eight heads of a sample
// at a time: their rows lie next to one another and share cache lines and pages (64 tokens x 8 heads over ragged caches:
// 124 us one by one, 114 by eights), while the samples, long and short, spread over the XCDs (135 us in eight runs).  Few
// pairs are cut into eight runs of tiles, so that no XCD gets a pair more than another.
struct Unit {
    int pair, tile, split;
};
__device__ __forceinline__ Unit unit_of(const AttnArgs& a) {
    const unsigned id = (unsigned)rs_block_id(), x = id & 7, j = id >> 3, splits = a.splits, per_pair = a.tiles * splits;
    const unsigned pairs = (unsigned)a.B * a.Hk;
    unsigned pair, in;
    if (a.dealt) {
        const unsigned per_deal = per_pair * a.dealt, k = j / per_deal, rest = j - k * per_deal;
        pair = (k * 8 + x) * a.dealt + rest / per_pair;
        in = rest % per_pair;
    } else {
        const unsigned run = (pairs * per_pair + 7) / 8, unit = x * run + j;
        pair = j < run ? unit / per_pair : pairs;
        in = unit % per_pair;
    }
    if (pair >= pairs) return {-1, 0, 0};
    return {(int)pair, (int)(in / splits), (int)(in % splits)};
}
inline long long order_units(AttnArgs& a) {      // the workgroups to launch for a.tiles and a.splits
    const long long pairs = (long long)a.B * a.Hk, per_pair = (long long)a.tiles * a.splits;
    int g = 1;
    while (g < 8 && a.Hk % (2 * g) == 0 && pairs / (2 * g) >= 64) g *= 2;
    a.dealt = pairs / g >= 64 || pairs % 8 == 0 ? g : 0;
    return a.dealt ? (pairs + 8 * g - 1) / (8 * g) * (8 * g) * per_pair : (pairs * per_pair + 7) / 8 * 8;
}

template <typename T, int DP> constexpr int tile_rows() { return sizeof(T) == 4 && DP == 128 ? 32 : 64; }

// ---- forward -----------------------------------------------------------------------------------------------------
template <typename T, int DP, int NW, int KT, bool VEC>
__global__ __launch_bounds__(NW * 64) void attention_fwd_kernel(const AttnArgs a) {
    constexpr int NT = NW * 64, BM = NW * 32, CK = Mma<T>::CK, E = Mma<T>::E, NC = DP / CK, NB = DP / 32, KB = KT / 32;
    typedef typename Mma<T>::V V;
    typedef Tile<T, DP> L;
    __shared__ __align__(1024) T s_k[2][KT * DP];
    __shared__ __align__(1024) T s_v[2][KT * DP];
    const Unit unit = unit_of(a);
    if (unit.pair < 0) return;
    const int tile = a.tiles - 1 - unit.tile, split = unit.split;          // causal: the long rows first
    const int pair = unit.pair, b = pair / a.Hk, hk = pair % a.Hk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int rows = a.Tq * a.G, row = tile * BM + wave * 32 + (lane & 31);
    const int i = (unsigned)row / (unsigned)a.G, h = hk * a.G + (unsigned)row % (unsigned)a.G;
    const bool live = row < rows;
    const int lim = live ? row_limit(a, b, i) : 0;
    // keys any row of the workgroup sees, and all live rows of this wave (rows only see more further down)
    const int last = min(tile * BM + BM, rows) - 1;
    int end = row_limit(a, b, last / a.G);
    if (end == 0) {                                               // its last rows may lie behind the sample's
        const int n = a.qlen ? min(a.qlen[b], a.Tq) : a.Tq;
        if (n > 0 && n - 1 < last / a.G && n - 1 >= tile * BM / a.G) end = row_limit(a, b, n - 1);
    }
    int low = lim;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) low = min(low, __shfl_xor(low, o, 64));
    low = __builtin_amdgcn_readfirstlane(low);
    int k0 = 0;
    if (a.splits > 1) {                                           // this share's whole tiles of them
        const int per = ((end + KT - 1) / KT + a.splits - 1) / a.splits * KT;
        k0 = min(split * per, end);
        end = min(k0 + per, end);
    }

    V qf[NC];
    {
        const T* qr = row_ptr<T>(a.q, b, live ? i : 0, live ? h : 0);
#pragma unroll
        for (int c = 0; c < NC; ++c) qf[c] = fetch<T, VEC>(qr, c * CK + half * E, a.D, live);     // whatever it holds where lim = 0
    }
    rs_f32x16 acc[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[n][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float scale2 = a.scale * LOG2E;
    const T* kp = row_ptr<T>(a.k, b, 0, hk);
    const T* vp = row_ptr<T>(a.v, b, 0, hk);
    Feed<T, DP, KT, NT, VEC> fk(a.k.t, a.D), fv(a.v.t, a.D);
    fk.seek(kp, k0, end);
    fv.seek(vp, k0, end);
    if (k0 < end) {
        fk.next(s_k[0]);
        fv.next(s_v[0]);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) settle(qf[c]);
    for (int buf = 0; k0 < end; k0 += KT, buf ^= 1) {
        fk.land(s_k[buf]);
        fv.land(s_v[buf]);
        feed_sync<VEC>();      // the other buffer's readers are past it, too
        if (k0 + KT < end) {
            fk.next(s_k[buf ^ 1]);
            fv.next(s_v[buf ^ 1]);
        }
        rs_f32x16 s[KB];
#pragma unroll
        for (int n = 0; n < KB; ++n) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[n][e] = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c) s[n] = Mma<T>::mul(L::rows(s_k[buf], n * 32, c), qf[c], s[n]);
        }
        if (k0 + KT > low) {
#pragma unroll
            for (int n = 0; n < KB; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (k0 + n * 32 + reg_row(e) >= lim) s[n][e] = -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int n = 0; n < KB; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, s[n][e]);
        top = half_max(top) * scale2;
        const float m_new = fmaxf(m, top);
        const float base = m_new == -INFINITY ? 0.f : m_new;     // nothing seen yet: exp2(-inf - 0) = 0 throughout
        const float alpha = __builtin_amdgcn_exp2f(m - base);
        m = m_new;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < KB; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[n][e] = __builtin_amdgcn_exp2f(s[n][e] * scale2 - (base - P_SHIFT<T>));
                sum += s[n][e];
            }
        l = l * alpha + sum;                                      // this half's keys only
        if (__any(alpha != 1.f)) {
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[n][e] *= alpha;
        }
#pragma unroll
        for (int n = 0; n < KB; ++n)
#pragma unroll
            for (int c = 0; c < 32 / CK; ++c) {
                const V p = pack<T>(s[n], c);
#pragma unroll
                for (int d = 0; d < NB; ++d) acc[d] = Mma<T>::mul(L::cols(s_v[buf], n * 32 + c * CK, d * 32), p, acc[d]);
            }
    }
    if (!live) return;
    l = half_sum(l);
    const bool none = l == 0.f;                                   // nothing seen: zeros, whatever the other rows' keys hold
    const float inv = 1.f / l;
    if (a.splits > 1) {
        const long long at = ((long long)split * a.B * a.Hk + pair) * rows + row;
        if (half == 0) a.part_ml[at] = none ? -INFINITY : m + log2f(l) - P_SHIFT<T>;
#pragma unroll
        for (int d = 0; d < NB; ++d)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                float o[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) o[x] = none ? 0.f : acc[d][e + x] * inv;
                store4<float>(a.part_o + at * a.D, d * 32 + reg_row(e), a.D, a.D % 4 == 0, o);
            }
        return;
    }
    if (a.lse && half == 0) a.lse[((long long)b * a.Hk * a.G + h) * a.Tq + i] = none ? -INFINITY : (m + log2f(l) - P_SHIFT<T>) * LN2;
    T* out = (T*)a.out + (((long long)b * a.Tq + i) * a.Hk * a.G + h) * a.D;
#pragma unroll
    for (int d = 0; d < NB; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            float o[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) o[x] = none ? 0.f : acc[d][e + x] * inv;
            store4<T>(out, d * 32 + reg_row(e), a.D, a.out_vec, o);
        }
}

// At most 16 rows (single tokens, short chunks) in fp32, whose matrix instructions are slow enough to matter here: 16x16 tiles
// do half the work of 32x32 ones padded from 16 columns (531 samples x 4 rows x 2 heads of 96 on one key head over caches of up
// to 7632: 1155 -> 481 us, 3.2 TB/s; 64 tokens x 8 heads of 128 over 4096 keys each 385..420 us, 5.1 TB/s and up).  One wave, 16 or 32 keys at
// a time; as above otherwise.
template <int DP, int KT, bool VEC>
__global__ __launch_bounds__(64) void attention_few_fwd_kernel(const AttnArgs a) {
    typedef float T;
    constexpr int CK = Mma16<T>::CK, E = Mma16<T>::E, NC = DP / CK, ND = DP / 16, NK = KT / 16;
    typedef typename Mma16<T>::V V;
    typedef Tile<T, DP> L;
    __shared__ __align__(1024) T s_k[2][KT * DP];
    __shared__ __align__(1024) T s_v[2][KT * DP];
    const Unit unit = unit_of(a);
    if (unit.pair < 0) return;
    const int split = unit.split, pair = unit.pair, b = pair / a.Hk, hk = pair % a.Hk;
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int rows = a.Tq * a.G, i = (unsigned)col / (unsigned)a.G, h = hk * a.G + (unsigned)col % (unsigned)a.G;
    const bool live = col < rows;
    const int lim = live ? row_limit(a, b, i) : 0;
    int end = lim, low = lim;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
        end = max(end, __shfl_xor(end, o, 64));
        low = min(low, __shfl_xor(low, o, 64));
    }
    end = __builtin_amdgcn_readfirstlane(end);
    low = __builtin_amdgcn_readfirstlane(low);
    int k0 = 0;
    if (a.splits > 1) {
        const int per = ((end + KT - 1) / KT + a.splits - 1) / a.splits * KT;
        k0 = min(split * per, end);
        end = min(k0 + per, end);
    }
    V qf[NC];
    const T* qr = row_ptr<T>(a.q, b, live ? i : 0, live ? h : 0);
#pragma unroll
    for (int c = 0; c < NC; ++c) qf[c] = fetch<T, VEC>(qr, c * CK + g * E, a.D, lim > 0);
    rs_f32x4 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = rs_f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const float scale2 = a.scale * LOG2E;
    Feed<T, DP, KT, 64, VEC> fk(a.k.t, a.D), fv(a.v.t, a.D);
    fk.seek(row_ptr<T>(a.k, b, 0, hk), k0, end);
    fv.seek(row_ptr<T>(a.v, b, 0, hk), k0, end);
    if (k0 < end) {
        fk.next(s_k[0]);
        fv.next(s_v[0]);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) settle(qf[c]);
    for (int buf = 0; k0 < end; k0 += KT, buf ^= 1) {
        fk.land(s_k[buf]);
        fv.land(s_v[buf]);
        feed_sync<VEC>();
        if (k0 + KT < end) {
            fk.next(s_k[buf ^ 1]);
            fv.next(s_v[buf ^ 1]);
        }
        rs_f32x4 s[NK];
        float top = -INFINITY;
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            s[n] = rs_f32x4{0.f, 0.f, 0.f, 0.f};
            const int r = n * 16 + col;
#pragma unroll
            for (int c = 0; c < NC; ++c)
                s[n] = Mma16<T>::mul(*(const V*)(s_k[buf] + r * DP + ((c * 4 + g) ^ L::swz(r)) * E), qf[c], s[n]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (k0 + KT > low && k0 + n * 16 + 4 * g + e >= lim) s[n][e] = -INFINITY;
                top = fmaxf(top, s[n][e]);
            }
        }
        const float m_new = fmaxf(m, col_max(top) * scale2), base = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m - base);
        m = m_new;
        l *= alpha;                                               // this lane's keys only
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[n][e] = __builtin_amdgcn_exp2f(s[n][e] * scale2 - base);
                l += s[n][e];
            }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[d][e] *= alpha;
#pragma unroll
            for (int n = 0; n < NK; ++n) {
                V v;
                const int at = d * 16 + col;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int r = n * 16 + 4 * g + x;
                    v[x] = s_v[buf][r * DP + ((at / E) ^ L::swz(r)) * E + at % E];
                }
                acc[d] = Mma16<T>::mul(v, s[n], acc[d]);
            }
        }
    }
    l = col_sum(l);
    if (!live) return;
    const bool none = l == 0.f;
    const float inv = 1.f / l;
    const bool shared_out = a.splits > 1;
    const long long at = ((long long)split * a.B * a.Hk + pair) * rows + col;
    T* out = shared_out ? a.part_o + at * a.D : (T*)a.out + (((long long)b * a.Tq + i) * a.Hk * a.G + h) * a.D;
    if (g == 0) {
        if (shared_out) a.part_ml[at] = none ? -INFINITY : m + log2f(l);
        else if (a.lse) a.lse[((long long)b * a.Hk * a.G + h) * a.Tq + i] = none ? -INFINITY : (m + log2f(l)) * LN2;
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = none ? 0.f : acc[d][e] * inv;
        store4<T>(out, d * 16 + 4 * g, a.D, shared_out ? a.D % 4 == 0 : a.out_vec, x);
    }
}

// Joins the shares of a row: weights exp2(lse_s - max) over their sum.  32 lanes to a row: they fetch the statistics of all
// shares at once (at most 64), then four elements of each share apiece.
template <typename T> __global__ __launch_bounds__(256) void attention_join_kernel(const AttnArgs a) {
    const long long rows = (long long)a.Tq * a.G, all = rows * a.B * a.Hk;
    const long long at = rs_block_id() * 8 + (threadIdx.x >> 5);
    if (at >= all) return;
    const int lane = threadIdx.x & 31;
    const long long pair = at / rows;
    const int row = (int)(at - pair * rows), i = row / a.G, b = (int)(pair / a.Hk), h = (int)(pair % a.Hk) * a.G + row % a.G;
    const float l0 = lane < a.splits ? a.part_ml[lane * all + at] : -INFINITY;
    const float l1 = lane + 32 < a.splits ? a.part_ml[(lane + 32) * all + at] : -INFINITY;
    float m = fmaxf(l0, l1);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 32));
    const float base = m == -INFINITY ? 0.f : m, w0 = __builtin_amdgcn_exp2f(l0 - base), w1 = __builtin_amdgcn_exp2f(l1 - base);
    float l = w0 + w1;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor(l, o, 32);
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    const int d = lane * 4;
    const bool vec = a.D % 4 == 0;
    for (int s0 = 0; s0 < a.splits; s0 += 8) {                    // eight shares in flight
        float w[8], x[8][4];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int s = s0 + u;
            w[u] = s < a.splits ? __shfl(s < 32 ? w0 : w1, s & 31, 32) : 0.f;
            x[u][0] = x[u][1] = x[u][2] = x[u][3] = 0.f;
            if (s >= a.splits) continue;
            const float* p = a.part_o + (s * all + at) * a.D + d;
            if (vec && d < a.D) {
                *(rs_f32x4*)x[u] = *(const rs_f32x4*)p;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[u][e] = d + e < a.D ? p[e] : 0.f;
            }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += w[u] * x[u][e];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= inv;
    store4<T>((T*)a.out + (((long long)b * a.Tq + i) * a.Hk * a.G + h) * a.D, d, a.D, a.out_vec, o);
    if (a.lse && lane == 0) a.lse[((long long)b * a.Hk * a.G + h) * a.Tq + i] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
}

// ---- dq, and delta for the other gradients -----------------------------------------------------------------------------
template <typename T, int DP, int NW, bool VEC>
__global__ __launch_bounds__(NW * 64) void attention_dq_kernel(const AttnArgs a) {
    constexpr bool BOTH = sizeof(T) == 2 && DP <= 64, F16 = Mma<T>::F16;      // dS in two parts, see above; Range
    constexpr int KT = tile_rows<T, DP>();
    constexpr int NT = NW * 64, BM = NW * 32, CK = Mma<T>::CK, E = Mma<T>::E, NC = DP / CK, NB = DP / 32, KB = KT / 32;
    typedef typename Mma<T>::V V;
    typedef Tile<T, DP> L;
    __shared__ __align__(1024) T s_k[2][KT * DP];
    __shared__ __align__(1024) T s_v[2][KT * DP];
    const Unit unit = unit_of(a);
    if (unit.pair < 0) return;
    const int tile = a.tiles - 1 - unit.tile;
    const int pair = unit.pair, b = pair / a.Hk, hk = pair % a.Hk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int rows = a.Tq * a.G, row = tile * BM + wave * 32 + (lane & 31);
    const int i = (unsigned)row / (unsigned)a.G, h = hk * a.G + (unsigned)row % (unsigned)a.G;
    const bool live = row < rows;
    const int lim = live ? row_limit(a, b, i) : 0;
    const int last = min(tile * BM + BM, rows) - 1;
    int end = row_limit(a, b, last / a.G);
    if (end == 0) {
        const int n = a.qlen ? min(a.qlen[b], a.Tq) : a.Tq;
        if (n > 0 && n - 1 < last / a.G && n - 1 >= tile * BM / a.G) end = row_limit(a, b, n - 1);
    }
    int low = lim;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) low = min(low, __shfl_xor(low, o, 64));
    low = __builtin_amdgcn_readfirstlane(low);

    V qf[NC], gf[NC];
    float delta = 0.f, lse2 = INFINITY;
    Range range;                                                  // of the lane's row: its factor goes into lse2
    {
        const bool has = live && lim > 0;
        const T* qr = row_ptr<T>(a.q, b, live ? i : 0, live ? h : 0);
        const T* gr = row_ptr<T>(a.go, b, live ? i : 0, live ? h : 0);
        const T* orow = row_ptr<T>(a.o, b, live ? i : 0, live ? h : 0);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            qf[c] = fetch<T, VEC>(qr, c * CK + half * E, a.D, has);
            gf[c] = fetch<T, VEC>(gr, c * CK + half * E, a.D, has);
            const V of = fetch<T, VEC>(orow, c * CK + half * E, a.D, has);
#pragma unroll
            for (int e = 0; e < E; ++e) delta += (float)gf[c][e] * (float)of[e];
        }
        delta = half_sum(delta);
        const long long at = ((long long)b * a.Hk * a.G + h) * a.Tq + i;
        if (has) lse2 = back_lse(a.lse[at]);
        if (live && half == 0) a.delta[at] = delta;
    }
    rs_f32x16 acc[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[n][e] = 0.f;
    const float scale2 = a.scale * LOG2E;
    const T* kp = row_ptr<T>(a.k, b, 0, hk);
    const T* vp = row_ptr<T>(a.v, b, 0, hk);
    Feed<T, DP, KT, NT, VEC> fk(a.k.t, a.D), fv(a.v.t, a.D);
    fk.seek(kp, 0, end);
    fv.seek(vp, 0, end);
    if (0 < end) {
        fk.next(s_k[0]);
        fv.next(s_v[0]);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        settle(qf[c]);
        settle(gf[c]);
    }
    for (int k0 = 0, buf = 0; k0 < end; k0 += KT, buf ^= 1) {
        fk.land(s_k[buf]);
        fv.land(s_v[buf]);
        feed_sync<VEC>();      // the other buffer's readers are past it, too
        if (k0 + KT < end) {
            fk.next(s_k[buf ^ 1]);
            fv.next(s_v[buf ^ 1]);
        }
#pragma unroll
        for (int n = 0; n < KB; ++n) {
            rs_f32x16 s, dp;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                s = Mma<T>::mul(L::rows(s_k[buf], n * 32, c), qf[c], s);
                dp = Mma<T>::mul(L::rows(s_v[buf], n * 32, c), gf[c], dp);
            }
            if (k0 + n * 32 + 32 > low) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (k0 + n * 32 + reg_row(e) >= lim) s[e] = -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(s[e] * scale2 - lse2) * (dp[e] - delta);
            if constexpr (F16) {
                const float top = half_max(reg_max(s));
                if (__any(range.past(top))) {
                    const int by = range.follow(top);
                    lse2 -= (float)by;
                    scale_by(s, by);
#pragma unroll
                    for (int d = 0; d < NB; ++d) scale_by(acc[d], by);
                }
            }
#pragma unroll
            for (int c = 0; c < 32 / CK; ++c) {
                const V p = pack<T>(s, c);
#pragma unroll
                for (int d = 0; d < NB; ++d) {
                    const V kt = L::cols(s_k[buf], n * 32 + c * CK, d * 32);
                    acc[d] = Mma<T>::mul(kt, p, acc[d]);
                    if constexpr (BOTH) acc[d] = Mma<T>::mul(kt, pack_rest<T>(s, c, p), acc[d]);
                }
            }
        }
    }
    if (!live) return;
    T* out = (T*)a.dq + (((long long)b * a.Tq + i) * a.Hk * a.G + h) * a.D;
    const float back = a.scale * range.unit();
#pragma unroll
    for (int d = 0; d < NB; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            float o[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) o[x] = lse2 == INFINITY ? 0.f : acc[d][e + x] * back;      // saw nothing: zeros
            store4<T>(out, d * 32 + reg_row(e), a.D, a.out_vec, o);
        }
}

// ---- dk and dv -----------------------------------------------------------------------------------------------------------
template <typename T, int DP, int NW, bool VEC>
__global__ __launch_bounds__(NW * 64, DP == 128 && sizeof(T) == 2 && VEC && NW == 4 ? 2 : 1) void attention_dkv_kernel(const AttnArgs a) {
    constexpr bool BOTH = sizeof(T) == 2 && DP <= 64, F16 = Mma<T>::F16;      // dS in two parts, see above; Range
    constexpr bool VLDS = DP == 128 && sizeof(T) == 2;
    constexpr int RT = VLDS ? 32 : tile_rows<T, DP>();
    constexpr int NT = NW * 64, BN = NW * 32, CK = Mma<T>::CK, E = Mma<T>::E, NC = DP / CK, NB = DP / 32, RB = RT / 32;
    typedef typename Mma<T>::V V;
    typedef Tile<T, DP> L;
    __shared__ __align__(1024) T s_q[2][RT * DP];
    __shared__ __align__(1024) T s_g[2][RT * DP];
    __shared__ __align__(1024) T s_v[VLDS ? BN * DP : 1];
    __shared__ __align__(16) float s_lse[2][RT], s_delta[2][RT];
    const Unit unit = unit_of(a);
    if (unit.pair < 0) return;
    const int tile = unit.tile, split = unit.split;               // causal: the first keys are seen by the most rows
    const int pair = unit.pair, b = pair / a.Hk, hk = pair % a.Hk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int key = tile * BN + wave * 32 + (lane & 31);
    const int len = a.len ? min(max(a.len[b], 0), a.Tk) : a.Tk;
    const int qrows = a.qlen ? min(max(a.qlen[b], 0), a.Tq) : a.Tq;
    int begin = 0;                                                // first row that sees a key of this workgroup
    long long start = 0;
    if (a.causal) {
        start = a.qstart ? a.qstart[b] : a.start;
        const long long f = (long long)tile * BN - start;
        begin = f <= 0 ? 0 : f >= qrows ? qrows : (int)f;
    }
    const int stop = tile * BN < len ? qrows : 0;

    // a key that no row sees is none: zeros here and in the results, whatever it holds
    const bool has = key < len && qrows > 0 && (!a.causal || key <= start + qrows - 1);
    V kf[NC], vf[VLDS ? 1 : NC];
    {
        const T* kr = row_ptr<T>(a.k, b, has ? key : 0, hk);
        const T* vr = row_ptr<T>(a.v, b, has ? key : 0, hk);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            kf[c] = fetch<T, VEC>(kr, c * CK + half * E, a.D, has);
            if constexpr (!VLDS) vf[c] = fetch<T, VEC>(vr, c * CK + half * E, a.D, has);
        }
    }
    Range range;                                                  // of the lane's key
    float factor = 1.f;
    rs_f32x16 dk[NB], dv[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[n][e] = dv[n][e] = 0.f;
    const float scale2 = a.scale * LOG2E;
    Feed<T, DP, RT, NT, VEC> fq(a.q.t, a.D), fg(a.go.t, a.D);
    // a turn is a row tile of one head of the group; this workgroup takes its share of them, the loads run one ahead
    const int per_head = begin < stop ? (stop - begin + RT - 1) / RT : 0, all = per_head * a.G;
    const int share = (all + a.splits - 1) / a.splits, turn0 = min(split * share, all), turns = min(turn0 + share, all) - turn0;
    int h = hk * a.G, r_next = begin;
    if (turns > 0) {
        h += turn0 / per_head;
        r_next += turn0 % per_head * RT;
        fq.seek(row_ptr<T>(a.q, b, 0, h), r_next, stop);
        fg.seek(row_ptr<T>(a.go, b, 0, h), r_next, stop);
        if constexpr (VLDS) {            // (without a turn nothing would wait for it)
            Feed<T, DP, BN, NT, VEC> fv(a.v.t, a.D);
            fv.seek(row_ptr<T>(a.v, b, 0, hk), tile * BN, (int)min(a.causal ? start + qrows : len, (long long)len));
            fv.next(s_v);
            fv.land(s_v);
        }
    }
    int r0 = r_next;
    float r_lse, r_delta;
    auto load = [&](int buf) {
        // all lanes, a valid row each, and used only when the tile has landed: a wait for these would wait for the tile
        const long long at = ((long long)b * a.Hk * a.G + h) * a.Tq + min(r_next + (int)(threadIdx.x % RT), stop - 1);
        r_lse = a.lse[at];
        r_delta = a.delta[at];
        fq.next(s_q[buf]);
        fg.next(s_g[buf]);
        if ((r_next += RT) >= stop && ++h < (hk + 1) * a.G) {
            r_next = begin;
            fq.seek(row_ptr<T>(a.q, b, 0, h), begin, stop);
            fg.seek(row_ptr<T>(a.go, b, 0, h), begin, stop);
        }
    };
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        settle(kf[c]);
        if constexpr (!VLDS) settle(vf[c]);
    }
    if (turns > 0) load(0);
    for (int turn = 0, buf = 0; turn < turns; ++turn, buf ^= 1) {
        // a key that row r0 + x does not see: x < hide (selected below, not multiplied: it may hold anything)
        const long long ahead = (long long)key - start - r0;
        const int hide = !a.causal || ahead <= 0 ? 0 : ahead < RT ? (int)ahead : RT;
        fq.land(s_q[buf]);
        fg.land(s_g[buf]);
        // a row that sees nothing, or is none: exp2(z - inf) = 0
        asm volatile("" : "+v"(r_lse), "+v"(r_delta));            // all lanes wait for them here (see settle)
        if (threadIdx.x < RT) {
            s_lse[buf][threadIdx.x] = r0 + (int)threadIdx.x >= stop ? INFINITY : back_lse(r_lse) - P_SHIFT<T>;
            s_delta[buf][threadIdx.x] = r_delta;
        }
        feed_sync<VEC>();
        r0 = r_next;
        if (turn + 1 < turns) load(buf ^ 1);
#pragma unroll
        for (int n = 0; n < RB; ++n) {
            rs_f32x16 s, dp;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                s = Mma<T>::mul(L::rows(s_q[buf], n * 32, c), kf[c], s);
                V vc;
                if constexpr (VLDS) vc = L::rows(s_v, wave * 32, c);
                else vc = vf[c];
                dp = Mma<T>::mul(L::rows(s_g[buf], n * 32, c), vc, dp);
            }
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int r = n * 32 + reg_row(e);
                const rs_f32x4 ls = *(const rs_f32x4*)&s_lse[buf][r], de = *(const rs_f32x4*)&s_delta[buf][r];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float p = __builtin_amdgcn_exp2f(s[e + x] * scale2 - ls[x]);
                    s[e + x] = p;
                    dp[e + x] = p * (dp[e + x] - de[x]);
                }
            }
            if (__any(hide > n * 32)) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (n * 32 + reg_row(e) < hide) s[e] = dp[e] = 0.f;
            }
            if constexpr (F16) {
#pragma unroll
                for (int e = 0; e < 16; ++e) dp[e] *= factor;
                const float top = half_max(reg_max(dp));
                if (__any(range.past(top))) {
                    const int by = range.follow(top);
                    factor = ldexpf(factor, by);
                    scale_by(dp, by);
#pragma unroll
                    for (int d = 0; d < NB; ++d) scale_by(dk[d], by);
                }
            }
#pragma unroll
            for (int c = 0; c < 32 / CK; ++c) {
                const V p = pack<T>(s, c), ds = pack<T>(dp, c);
#pragma unroll
                for (int d = 0; d < NB; ++d) {
                    const V qt = L::cols(s_q[buf], n * 32 + c * CK, d * 32);
                    dv[d] = Mma<T>::mul(L::cols(s_g[buf], n * 32 + c * CK, d * 32), p, dv[d]);
                    dk[d] = Mma<T>::mul(qt, ds, dk[d]);
                    if constexpr (BOTH) dk[d] = Mma<T>::mul(qt, pack_rest<T>(dp, c, ds), dk[d]);
                }
            }
        }
    }
    if (key >= a.Tk) return;
    const long long at = (((long long)b * a.Tk + key) * a.Hk + hk) * a.D;
    const float back = a.scale * P_UNIT<T> * range.unit();
#pragma unroll
    for (int d = 0; d < NB; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            float o[4], u[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                o[x] = has ? dk[d][e + x] * back : 0.f;
                u[x] = has ? dv[d][e + x] * P_UNIT<T> : 0.f;
            }
            if (a.splits > 1) {
                const long long total = (long long)a.B * a.Tk * a.Hk * a.D;
                store4<float>(a.part_o + 2 * split * total + at, d * 32 + reg_row(e), a.D, a.D % 4 == 0, o);
                store4<float>(a.part_o + (2 * split + 1) * total + at, d * 32 + reg_row(e), a.D, a.D % 4 == 0, u);
            } else {
                store4<T>((T*)a.dk + at, d * 32 + reg_row(e), a.D, a.out_vec, o);
                store4<T>((T*)a.dv + at, d * 32 + reg_row(e), a.D, a.out_vec, u);
            }
        }
}

// dk and dv from the shares, added in their order.
template <typename T> __global__ __launch_bounds__(256) void attention_dkv_join_kernel(const AttnArgs a) {
    const long long total = (long long)a.B * a.Tk * a.Hk * a.D, at = (rs_block_id() * 256 + threadIdx.x) * 4;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        T* out = (T*)(w ? a.dv : a.dk);
        if (at + 4 <= total && a.out_vec) {
            rs_f32x4 x = *(const rs_f32x4*)(a.part_o + w * total + at);
            for (int s = 1; s < a.splits; ++s) x += *(const rs_f32x4*)(a.part_o + (2 * s + w) * total + at);
            const float o[4] = {x[0], x[1], x[2], x[3]};
            store4<T>(out + at, 0, 4, true, o);
        } else {
            for (long long i = at; i < at + 4 && i < total; ++i) {
                float x = 0.f;
                for (int s = 0; s < a.splits; ++s) x += a.part_o[(2 * s + w) * total + i];
                out[i] = (T)x;
            }
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
inline int padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }
inline int waves_for(long long rows) { return rows <= 32 ? 1 : rows <= 64 ? 2 : 4; }
inline int key_tile(int dtype, int D, int nw) { return nw == 1 || (dtype == RS_F32 && padded(D) == 128) ? 32 : 64; }     // at least

// Shares of the keys: few rows leave most of the chip idle, so the keys of a sample are split until there are about
// eight waves for every CU, but no share is shorter than four tiles.
int splits_for(int dtype, int B, int Tq, int Tk, int Hk, int G, int D) {
    const long long rows = (long long)Tq * G;
    const int nw = waves_for(rows);
    const long long units = (long long)B * Hk * ((rows + nw * 32 - 1) / (nw * 32));
    const long long want = 2048 / nw / units, most = Tk / (4 * key_tile(dtype, D, nw));
    const long long s = want < most ? want : most;
    return s < 1 ? 1 : s > 64 ? 64 : (int)s;
}

// Shares of the rows for dk and dv.  Even work: split until there are two workgroups for every CU.  A causal mask or lengths
// give the key tiles uneven work, and one workgroup per key tile leaves some CUs with twice the mean: split until there are
// four (causal or ragged, dk / dv with their join at two and at four workgroups: 2 x 8192 x 4 key heads of 128 1847, 1161 us; 16384
// x 2 of 128 1803, 1730; 2 x 4096 x 8 of 128 200, 147; 2 x 2048 x 4 of 128 143, 128; 4 x 2048 x 8 of 64 75, 70; of 32 51, 48;
// the join costs more than it gives for the shortest: 16 x 1000 x 4 of 64 39, 45, 4096 x 2 of 64 93, 102.  Without a mask as
// many tiles as the first takes 1.20 ms in one share, 1.34 in four).  No share is shorter than eight row tiles.
int dkv_splits(int B, int Tq, int Tk, int Hk, int G, int uneven) {
    const long long units = (long long)B * Hk * rs_cdiv(Tk, Tk <= 64 ? 64 : 128), turns = (long long)G * rs_cdiv(Tq, 64);
    const long long want = (uneven ? 1024 : 512) / units, most = turns / 8, s = want < most ? want : most;
    return s < 1 ? 1 : s > 16 ? 16 : (int)s;
}

// KT: keys at a time.
template <typename T, int DP, int NW, int KT> void launch_fwd_tiles(const AttnArgs& a, dim3 grid, hipStream_t stream) {
    if (a.vec) hipLaunchKernelGGL((attention_fwd_kernel<T, DP, NW, KT, true>), grid, dim3(NW * 64), 0, stream, a);
    else hipLaunchKernelGGL((attention_fwd_kernel<T, DP, NW, KT, false>), grid, dim3(NW * 64), 0, stream, a);
}
template <typename T, int DP, int NW> int launch_fwd(AttnArgs a, hipStream_t stream) {
    const dim3 grid = rs_grid(order_units(a));
    // Heads of 33..64 in 16 bits over long keys: 128 at a time give the wave four independent chains of products; heads of 128
    // have no registers for it, short samples too few tiles (1537 keys x 12 heads x 3 fp16: 64 at a time 47.6 us, 128 42.1; 1000
    // keys 34.8, 30.6; 800, causal, 35.6, 37.8; 600 30.1, 30.4; 400 52.0, 60.7; ragged histories of up to 200 50, 64 and of up
    // to 70 19.7, 26.7)
    constexpr bool WIDE = NW == 4 && DP == 64 && sizeof(T) == 2;
    if constexpr (NW == 1 && sizeof(T) == 4) {
        constexpr int FEW = DP == 128 ? 16 : 32;
        if (a.Tq * a.G > 16) launch_fwd_tiles<T, DP, NW, 32>(a, grid, stream);
        else if (a.vec) hipLaunchKernelGGL((attention_few_fwd_kernel<DP, FEW, true>), grid, dim3(64), 0, stream, a);
        else hipLaunchKernelGGL((attention_few_fwd_kernel<DP, FEW, false>), grid, dim3(64), 0, stream, a);
    } else if (WIDE && a.Tk >= 900) {
        launch_fwd_tiles<T, DP, NW, WIDE ? 128 : tile_rows<T, DP>()>(a, grid, stream);
    } else {
        launch_fwd_tiles<T, DP, NW, NW == 1 ? 32 : tile_rows<T, DP>()>(a, grid, stream);
    }
    RS_CHECK_LAUNCH("rs_attention_fwd");
    if (a.splits > 1) {
        hipLaunchKernelGGL((attention_join_kernel<T>), rs_grid(((long long)a.B * a.Hk * a.Tq * a.G + 7) / 8), dim3(256), 0, stream, a);
        RS_CHECK_LAUNCH("rs_attention_fwd");
    }
    return RS_OK;
}
template <typename T, int DP> int launch_fwd(const AttnArgs& a, int nw, hipStream_t stream) {
    return nw == 1 ? launch_fwd<T, DP, 1>(a, stream) : nw == 2 ? launch_fwd<T, DP, 2>(a, stream) : launch_fwd<T, DP, 4>(a, stream);
}
template <typename T> int launch_fwd(const AttnArgs& a, int nw, hipStream_t stream) {
    const int dp = padded(a.D);
    return dp == 32 ? launch_fwd<T, 32>(a, nw, stream) : dp == 64 ? launch_fwd<T, 64>(a, nw, stream) : launch_fwd<T, 128>(a, nw, stream);
}

template <typename T, int DP, int NW> int launch_dq(AttnArgs a, hipStream_t stream) {
    a.tiles = rs_cdiv((long long)a.Tq * a.G, NW * 32);
    a.splits = 1;                            // a row's keys are not shared out here
    const dim3 grid = rs_grid(order_units(a));
    if (a.vec) hipLaunchKernelGGL((attention_dq_kernel<T, DP, NW, true>), grid, dim3(NW * 64), 0, stream, a);
    else hipLaunchKernelGGL((attention_dq_kernel<T, DP, NW, false>), grid, dim3(NW * 64), 0, stream, a);
    RS_CHECK_LAUNCH("rs_attention_bwd");
    return RS_OK;
}
template <typename T, int DP, int NW> int launch_dkv(AttnArgs a, hipStream_t stream) {
    a.tiles = rs_cdiv(a.Tk, NW * 32);
    const dim3 grid = rs_grid(order_units(a));
    if (a.vec) hipLaunchKernelGGL((attention_dkv_kernel<T, DP, NW, true>), grid, dim3(NW * 64), 0, stream, a);
    else hipLaunchKernelGGL((attention_dkv_kernel<T, DP, NW, false>), grid, dim3(NW * 64), 0, stream, a);
    RS_CHECK_LAUNCH("rs_attention_bwd");
    if (a.splits > 1) {
        const long long quads = ((long long)a.B * a.Tk * a.Hk * a.D + 3) / 4;
        hipLaunchKernelGGL((attention_dkv_join_kernel<T>), rs_grid((quads + 255) / 256), dim3(256), 0, stream, a);
        RS_CHECK_LAUNCH("rs_attention_bwd");
    }
    return RS_OK;
}
template <typename T, int DP> int launch_bwd(const AttnArgs& a, hipStream_t stream) {
    int rc = RS_OK;
    if (a.Tq > 0) rc = (long long)a.Tq * a.G <= 64 ? launch_dq<T, DP, 2>(a, stream) : launch_dq<T, DP, 4>(a, stream);
    if (rc == RS_OK && a.Tk > 0) rc = a.Tk <= 64 ? launch_dkv<T, DP, 2>(a, stream) : launch_dkv<T, DP, 4>(a, stream);
    return rc;
}
template <typename T> int launch_bwd(const AttnArgs& a, hipStream_t stream) {
    const int dp = padded(a.D);
    return dp == 32 ? launch_bwd<T, 32>(a, stream) : dp == 64 ? launch_bwd<T, 64>(a, stream) : launch_bwd<T, 128>(a, stream);
}

bool shape_ok(const char* who, int dtype, int B, int Tq, int Tk, int Hq, int Hk, int D, float scale) {
    if (!(dtype == RS_F32 || dtype == RS_BF16 || dtype == RS_F16)) {
        rs_set_error("%s: type %d not served", who, dtype);
        return false;
    }
    if (B < 0 || Tq < 0 || Tk < 0 || Hk < 1 || Hq < Hk || Hq % Hk || D < 1 || D > 128) {
        rs_set_error("%s: bad shape B=%d Tq=%d Tk=%d Hq=%d Hk=%d D=%d (D <= 128, Hq a multiple of Hk)", who, B, Tq, Tk, Hq, Hk, D);
        return false;
    }
    if (!(scale > 0.f) || scale > 1e30f) {
        rs_set_error("%s: scale must be positive and finite", who);
        return false;
    }
    // rows and workgroups are counted in 32 bits
    if ((long long)Tq * (Hq / Hk) > (1 << 30) || Tk > (1 << 30) || (long long)B * Hq * ((Tq > Tk ? Tq : Tk) / 32 + 1) > (1 << 30)) {
        rs_set_error("%s: too large", who);
        return false;
    }
    return true;
}

// An operand of T rows of D to a sample; the stride of a single row means nothing and becomes D.
AttnOperand operand(const void* p, long long b, long long t, long long h, int T, int D) { return {p, b, T > 1 ? t : D, h}; }
// 16-byte loads through a descriptor that ends with the last row: rows start at multiples of 16 bytes, do not overlap, and a
// tile of them stays within 31 bits.
bool operand_vec(const AttnOperand& x, int dtype, int D) {
    const int e = 16 / rs_elem_bytes(dtype);
    return !x.p || (rs_aligned16(x.p) && x.b % e == 0 && x.h % e == 0 && x.t % e == 0 && x.t >= D && x.t < (1 << 22));
}

}  // namespace

extern "C" {

size_t rs_attention_fwd_workspace_floats(int dtype, int B, int Tq, int Tk, int Hq, int Hk, int D) {
    if (B <= 0 || Tq <= 0 || Tk <= 0 || Hk < 1 || Hq < Hk || Hq % Hk || D < 1 || D > 128) return 0;
    if (rs_attention_small_ok(dtype, Tq, Tk, D)) return 0;
    const int s = splits_for(dtype, B, Tq, Tk, Hk, Hq / Hk, D);
    return s == 1 ? 0 : (size_t)s * B * Tq * Hq * (D + 1);
}

int rs_attention_fwd(int dtype, const void* q, long long qb, long long qt, long long qh, const void* k, long long kb, long long kt,
                     long long kh, const void* v, long long vb, long long vt, long long vh, int B, int Tq, int Tk, int Hq, int Hk,
                     int D, const int* lengths, const int* query_lengths, int causal, const int* query_starts, int query_start,
                     float scale, void* o, float* lse, float* workspace, size_t workspace_floats, rs_stream_t stream) {
    if (!shape_ok("rs_attention_fwd", dtype, B, Tq, Tk, Hq, Hk, D, scale)) return RS_ERR_ARG;
    if (B == 0 || Tq == 0) return RS_OK;
    RS_CHECK_ARG(q && o && (Tk == 0 || (k && v)), "rs_attention_fwd: null argument");
    AttnArgs a = {};
    a.q = operand(q, qb, qt, qh, Tq, D);
    a.k = operand(k, kb, kt, kh, Tk, D);
    a.v = operand(v, vb, vt, vh, Tk, D);
    a.out = o;
    a.lse = lse;
    a.len = lengths;
    a.qlen = query_lengths;
    a.qstart = query_starts;
    a.B = B, a.Tq = Tq, a.Tk = Tk, a.Hk = Hk, a.G = Hq / Hk, a.D = D, a.causal = causal != 0, a.start = query_start;
    a.scale = scale;
    a.vec = D % (16 / rs_elem_bytes(dtype)) == 0 && operand_vec(a.q, dtype, D) && operand_vec(a.k, dtype, D) && operand_vec(a.v, dtype, D);
    a.out_vec = D % 4 == 0 && rs_aligned16(o);
    if (rs_attention_small_ok(dtype, Tq, Tk, D)) return rs_attention_small_fwd(dtype, a, stream);
    const long long rows = (long long)Tq * a.G;
    const int nw = waves_for(rows);
    a.tiles = rs_cdiv(rows, nw * 32);
    a.splits = Tk > 0 ? splits_for(dtype, B, Tq, Tk, Hk, a.G, D) : 1;
    if (a.splits > 1) {
        const size_t need = rs_attention_fwd_workspace_floats(dtype, B, Tq, Tk, Hq, Hk, D);
        if (!workspace || workspace_floats < need) {
            rs_set_error("rs_attention_fwd: workspace of %zu floats, %zu needed", workspace_floats, need);
            return RS_ERR_WORKSPACE;
        }
        RS_CHECK_ARG(rs_aligned16(workspace), "rs_attention_fwd: workspace must be aligned to 16 bytes");
        a.part_o = workspace;
        a.part_ml = workspace + (size_t)a.splits * B * Tq * Hq * D;
    }
    if (dtype == RS_F32) return launch_fwd<float>(a, nw, stream);
    if (dtype == RS_BF16) return launch_fwd<__bf16>(a, nw, stream);
    return launch_fwd<_Float16>(a, nw, stream);
}

size_t rs_attention_bwd_workspace_floats(int dtype, int B, int Tq, int Tk, int Hq, int Hk, int D, int uneven) {
    if (B <= 0 || Tq <= 0 || Tk < 0 || Hk < 1 || Hq < Hk || Hq % Hk || D < 1 || D > 128) return 0;
    if (rs_attention_small_ok(dtype, Tq, Tk, D)) return 0;
    const int s = Tk > 0 ? dkv_splits(B, Tq, Tk, Hk, Hq / Hk, uneven) : 1;
    // delta, up to a multiple of four floats, then the shares of dk and dv
    return ((size_t)B * Tq * Hq + 3) / 4 * 4 + (s > 1 ? (size_t)2 * s * B * Tk * Hk * D : 0);
}

int rs_attention_bwd(int dtype, const void* go, long long gb, long long gt, long long gh, const void* q, long long qb, long long qt,
                     long long qh, const void* k, long long kb, long long kt, long long kh, const void* v, long long vb,
                     long long vt, long long vh, const void* o, long long ob, long long ot, long long oh, const float* lse, int B,
                     int Tq, int Tk, int Hq, int Hk, int D, const int* lengths, const int* query_lengths, int causal,
                     const int* query_starts, int query_start, float scale, void* dq, void* dk, void* dv, float* workspace,
                     size_t workspace_floats, rs_stream_t stream) {
    if (!shape_ok("rs_attention_bwd", dtype, B, Tq, Tk, Hq, Hk, D, scale)) return RS_ERR_ARG;
    if (B == 0 || (Tq == 0 && Tk == 0)) return RS_OK;
    RS_CHECK_ARG((Tq == 0 || (go && q && o && lse && dq)) && (Tk == 0 || (k && v && dk && dv)), "rs_attention_bwd: null argument");
    const int uneven = causal != 0 || lengths || query_lengths;
    const size_t need = rs_attention_bwd_workspace_floats(dtype, B, Tq, Tk, Hq, Hk, D, uneven);
    if (need && (!workspace || workspace_floats < need)) {
        rs_set_error("rs_attention_bwd: workspace of %zu floats, %zu needed", workspace_floats, need);
        return RS_ERR_WORKSPACE;
    }
    RS_CHECK_ARG(rs_aligned16(workspace), "rs_attention_bwd: workspace must be aligned to 16 bytes");
    AttnArgs a = {};
    a.q = operand(q, qb, qt, qh, Tq, D);
    a.k = operand(k, kb, kt, kh, Tk, D);
    a.v = operand(v, vb, vt, vh, Tk, D);
    a.o = operand(o, ob, ot, oh, Tq, D);
    a.go = operand(go, gb, gt, gh, Tq, D);
    a.dq = dq, a.dk = dk, a.dv = dv;
    a.lse = (float*)lse;
    a.delta = workspace;
    a.len = lengths;
    a.qlen = query_lengths;
    a.qstart = query_starts;
    a.B = B, a.Tq = Tq, a.Tk = Tk, a.Hk = Hk, a.G = Hq / Hk, a.D = D, a.causal = causal != 0, a.start = query_start;
    a.scale = scale;
    a.splits = Tq > 0 && Tk > 0 ? dkv_splits(B, Tq, Tk, Hk, a.G, uneven) : 1;
    a.part_o = workspace + ((size_t)B * Tq * Hq + 3) / 4 * 4;
    a.vec = D % (16 / rs_elem_bytes(dtype)) == 0 && operand_vec(a.q, dtype, D) && operand_vec(a.k, dtype, D) && operand_vec(a.v, dtype, D) &&
            operand_vec(a.o, dtype, D) && operand_vec(a.go, dtype, D);
    a.out_vec = D % 4 == 0 && rs_aligned16(dq) && rs_aligned16(dk) && rs_aligned16(dv);
    if (rs_attention_small_ok(dtype, Tq, Tk, D)) return rs_attention_small_bwd(dtype, a, stream);
    if (dtype == RS_F32) return launch_bwd<float>(a, stream);
    if (dtype == RS_BF16) return launch_bwd<__bf16>(a, stream);
    return launch_bwd<_Float16>(a, stream);
}

}  // extern "C"
