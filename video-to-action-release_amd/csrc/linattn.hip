// Linear attention with a decay for each head:  S_t = a_t S_{t-1} + k_t v_t^T (fp32, Dk x Dv),  a_t = exp(g_t),  o_t = scale * S_t^T q_t.
// Whole sequences (v2a_linattn_fwd / v2a_linattn_bwd) and single tokens on a pool of states (v2a_linattn_step).
#include "common.h"
#include <type_traits>

namespace {

constexpr int LA_DMAX = 128;            // largest head width
constexpr float LA_GMIN = -1000.f;      // decays below exp(-1000) are 0 in fp32 already; the clamp makes -inf (a reset) ordinary arithmetic

template <int DT> struct LaT;           // element types: 0 fp32, 1 bf16, 2 fp16; in the chunked kernels also 3: fp32 computed in bf16 planes
template <> struct LaT<0> { typedef float T; static __device__ __forceinline__ float ld(float x) { return x; } static __device__ __forceinline__ float st(float x) { return x; } };
template <> struct LaT<3> : LaT<0> {};
template <> struct LaT<1> { typedef unsigned short T; static __device__ __forceinline__ float ld(T x) { return v2a_h2f<false>(x); } static __device__ __forceinline__ T st(float x) { return v2a_f2h<false>(x); } };
template <> struct LaT<2> { typedef unsigned short T; static __device__ __forceinline__ float ld(T x) { return v2a_h2f<true>(x); } static __device__ __forceinline__ T st(float x) { return v2a_f2h<true>(x); } };

struct LaArgs {
    const void *q, *k, *v, *dout;
    const float *g, *state;
    const int* lens;
    long long qs[3], ks[3], vs[3], gs[3], ds[3];       // element strides over (batch, token, head)
    int B, T, H, Hq, Hk, Hv, Dk, Dv;
    float scale;
};

__device__ __forceinline__ int la_len(const LaArgs& a, int b) {
    if (!a.lens) return a.T;
    const int n = a.lens[b];
    return n < 0 ? 0 : n > a.T ? a.T : n;
}
__device__ __forceinline__ float la_clampg(float g) { return g < LA_GMIN ? LA_GMIN : g; }

// ---------------------------------------------------------------------------------------------------------------------- chunked form
// A chunk is 64 tokens.  With G_i = g_1 + .. + g_i inside it, W_ij = exp(G_i - G_j) for j <= i and S the state before it,
//     o_i = scale (exp(G_i) S^T q_i + sum_j W_ij (q_i . k_j) v_j),      S' = exp(G_64) S + sum_j exp(G_64 - G_j) k_j v_j^T,
// all of it matrix products.  They run on 16 x 16 x 32 MFMA tiles whose 32-long reduction index is numbered so that no operand is ever
// shuffled; lane group g = lane / 16 holds eight slots of it.  Over tokens, slots 0 .. 3 are tokens 4 g .. of the first 16 and slots 4 .. 7
// those of the second 16: two stacked 16 x 16 score accumulators ARE the operand of the product with v, and two transposing LDS reads
// (ds_read_b64_tr_b16) of a row-major tile give the operand of the transposed tile.  Over a head's width the slots are eight neighbours
// 8 g ..: one 16-byte read of a row; the state's rows are dealt to its accumulators so that two of them are such an operand as well.
// Number formats: bf16 inputs are one exact 8-bit plane, fp16 inputs two (8 + 3 bits, exact); factors computed in fp32 (scores, states)
// are fed as two planes (off by at most 2^-17 of the value), decay-weighted values of the state update as three (exact fp32), because the
// state is an fp32 result and lives long.  Sums are fp32.  fp32 inputs are three planes in LDS, fp32 factors too, and a product is the six
// plane products of 2^-16 and more (each dropped one is below 2^-24 of it): 96 cycles of the matrix unit against 256 of the fp32 MFMA.  Where
// planes cost the second workgroup on a CU (heads up to 64 wide) or do not fit at all (the four tiles of the gradient), tiles stay fp32 and the
// fp32 MFMA (16 x 16 x 4) takes them in the same slot order.
// Running log decays are summed in fp64 and kept as a float pair: W of two tokens behind a reset (g clamped at -1000) keeps its digits.
constexpr int LA_C = 64;
#define LA_FENCE __builtin_amdgcn_sched_barrier(0)      // between stages: moved up, the next one's operands fill the registers
typedef __attribute__((ext_vector_type(4))) unsigned int la_u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned int la_u32x2;
typedef __attribute__((ext_vector_type(4))) __bf16 la_bf16x4;
typedef __attribute__((address_space(3))) la_bf16x4 la_lds_bf16x4;

template <int NP> struct LaP { la_u32x4 p[NP]; };      // eight values as NP bf16 planes
struct LaF { float x[8]; };                            // eight fp32 values
template <int DT> struct LaOp {                        // operands: of an input tile, of a score or state, of a weighted value
    static constexpr int NP = DT;
    typedef LaP<NP> In;
    typedef LaP<DT == 3 ? 3 : 2> C2;
    typedef LaP<3> C3;
};
template <int DT> constexpr bool la_f32() { return DT == 0 || DT == 3; }      // element type
template <> struct LaOp<0> {
    typedef LaF In;
    typedef LaF C2;
    typedef LaF C3;
    static constexpr int NP = 1;
};

template <int NP> __device__ __forceinline__ void la_split(const float* x, LaP<NP>& o) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float a = x[2 * e], b = x[2 * e + 1];
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const unsigned int h = v2a_pack_bf16x2(a, b);
            o.p[n][e] = h;
            a -= __uint_as_float(h << 16);
            b -= __uint_as_float(h & 0xffff0000u);
        }
    }
}
__device__ __forceinline__ void la_split(const float* x, LaF& o) {
#pragma unroll
    for (int e = 0; e < 8; ++e) o.x[e] = x[e];
}
template <int NP> __device__ __forceinline__ void la_join(const LaP<NP>& o, float* x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[2 * e] = __uint_as_float(o.p[NP - 1][e] << 16);
        x[2 * e + 1] = __uint_as_float(o.p[NP - 1][e] & 0xffff0000u);
#pragma unroll
        for (int n = NP - 2; n >= 0; --n) {
            x[2 * e] += __uint_as_float(o.p[n][e] << 16);
            x[2 * e + 1] += __uint_as_float(o.p[n][e] & 0xffff0000u);
        }
    }
}
__device__ __forceinline__ void la_join(const LaF& o, float* x) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = o.x[e];
}

// c[row: index of a][col: index of b] += sum over the 32 slots; small products first.  ALL: every pair of planes (both operands exact), else
// those at least as large as the pieces that the more finely split operand still holds
template <int NA, int NB, bool ALL = false> __device__ __forceinline__ void la_mma(f32x4& c, const LaP<NA>& a, const LaP<NB>& b) {
    constexpr int TOP = ALL ? NA + NB - 2 : (NA > NB ? NA : NB) - 1;
#pragma unroll
    for (int o = TOP; o >= 0; --o)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (o - i >= 0 && o - i < NB)
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v2a_bf16x8, a.p[i]), __builtin_bit_cast(v2a_bf16x8, b.p[o - i]), c, 0, 0, 0);
}
template <int A = 0, int B = 0, bool ALL = false> __device__ __forceinline__ void la_mma(f32x4& c, const LaF& a, const LaF& b) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x[e], b.x[e], c, 0, 0, 0);
}
template <int DT> __device__ __forceinline__ void la_mma_in(f32x4& c, const typename LaOp<DT>::In& a, const typename LaOp<DT>::In& b) {
    if constexpr (DT == 0) la_mma(c, a, b);
    else la_mma<LaOp<DT>::NP, LaOp<DT>::NP, DT != 3>(c, a, b);
}

// A 64 x D tile in LDS, rows padded by 16 bytes.  nat: lane % 16 = row, slots along the row; tr: lane % 16 = column, slots down the rows
template <int DT, int D> struct LaTile {
    static constexpr int NP = LaOp<DT>::NP;
    static constexpr int PITCH = DT == 0 ? (D + 4) * 4 : (D + 8) * 2;      // bytes
    static constexpr int PLANE = LA_C * PITCH;
    static constexpr int BYTES = PLANE * NP;
    static __device__ __forceinline__ void nat(const char* t, int row0, int kk, int lane, typename LaOp<DT>::In& o) {
        const char* q = t + (row0 + (lane & 15)) * PITCH + (kk * 32 + (lane >> 4) * 8) * (DT == 0 ? 4 : 2);
        if constexpr (DT == 0) {
            const float4 a = *(const float4*)q, b = *(const float4*)(q + 16);
            o.x[0] = a.x; o.x[1] = a.y; o.x[2] = a.z; o.x[3] = a.w; o.x[4] = b.x; o.x[5] = b.y; o.x[6] = b.z; o.x[7] = b.w;
        } else {
#pragma unroll
            for (int n = 0; n < NP; ++n) o.p[n] = *(const la_u32x4*)(q + n * PLANE);
        }
    }
    // lane % 16 = column col0 + CS (lane % 16 / 4) + lane % 4: 16 neighbours (CS 4), or every other four of 32 (CS 8)
    template <int CS> static __device__ __forceinline__ void tr(const char* t, int ks, int col0, int lane, typename LaOp<DT>::In& o) {
        if constexpr (DT == 0) {
            const char* q = t + (ks * 32 + (lane >> 4) * 4) * PITCH + (col0 + CS * ((lane & 15) >> 2) + (lane & 3)) * 4;
#pragma unroll
            for (int e = 0; e < 8; ++e) o.x[e] = *(const float*)(q + (e < 4 ? e : 12 + e) * PITCH);
        } else {
            const char* q = t + (ks * 32 + (lane >> 4) * 4 + ((lane & 15) >> 2)) * PITCH + (col0 + CS * (lane & 3)) * 2;
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                const la_u32x2 a = __builtin_bit_cast(la_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((la_lds_bf16x4*)(q + n * PLANE)));
                const la_u32x2 b = __builtin_bit_cast(la_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((la_lds_bf16x4*)(q + n * PLANE + 16 * PITCH)));
                o.p[n] = la_u32x4{a[0], a[1], b[0], b[1]};
            }
        }
    }
    static __device__ __forceinline__ void four(const char* t, int row, int col, float* x) {      // four neighbours of a row
        const char* q = t + row * PITCH;
        if constexpr (DT == 0) {
            const float4 a = *(const float4*)(q + col * 4);
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        } else {
            const la_u32x2 z = *(const la_u32x2*)(q + (NP - 1) * PLANE + col * 2);
            x[0] = __uint_as_float(z[0] << 16); x[1] = __uint_as_float(z[0] & 0xffff0000u);
            x[2] = __uint_as_float(z[1] << 16); x[3] = __uint_as_float(z[1] & 0xffff0000u);
#pragma unroll
            for (int n = NP - 2; n >= 0; --n) {
                const la_u32x2 a = *(const la_u32x2*)(q + n * PLANE + col * 2);
                x[0] += __uint_as_float(a[0] << 16); x[1] += __uint_as_float(a[0] & 0xffff0000u);
                x[2] += __uint_as_float(a[1] << 16); x[3] += __uint_as_float(a[1] & 0xffff0000u);
            }
        }
    }
};

// A value that is the same in all lanes, cut off from where it came from: what is computed from it is computed here and now.  Hoisted out of the
// chunk loop, the row offsets of all operands together overflow the scalar registers, whose spills take vector registers and instructions.
template <typename T> __device__ __forceinline__ T la_here(T x) {
    asm volatile("" : "+s"(x));
    return x;
}
template <typename T> __device__ __forceinline__ T* la_at(const void* base, unsigned off) { return (T*)((char*)base + off); }

// Global rows -> registers (load) -> LDS (store), so that the next chunk's rows are under way while this one is computed.  Rows from nv on
// and columns from Dx on are zeros and not read.  vec: base, strides and Dx allow 16-byte loads; else element by element.
template <int DT, int D, int NTH> struct LaLoad {
    typedef typename LaT<DT>::T E;
    static constexpr int EPC = la_f32<DT>() ? 4 : 8, CPR = D / EPC, N = LA_C * CPR / NTH;
    static_assert(LA_C * CPR % NTH == 0, "whole 16-byte pieces per thread");
    static_assert(NTH % CPR == 0, "a thread's pieces share their columns");
    la_u32x4 r[N];
    // Thread t owns columns EPC (t % CPR) .. of rows t / CPR + i NTH / CPR.  p is the same in all lanes: with the lane's part of the address in
    // 32 bits (which `vec` vouches for) the rest stays in scalar registers.
    __device__ __forceinline__ void load(const E* p, long long st_, int nv_, int Dx, int vec) {
        const long long st = la_here(st_);
        const int nv = la_here(nv_);
        const int row = threadIdx.x / CPR, c = (threadIdx.x % CPR) * EPC;
        const unsigned off = ((unsigned)row * (unsigned)st + (unsigned)c) * (unsigned)sizeof(E);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            r[i] = la_u32x4{0u, 0u, 0u, 0u};
            if (row + i * (NTH / CPR) < nv && c < Dx) {
                const E* u = p + st * (i * (NTH / CPR));
                if (vec) r[i] = *la_at<la_u32x4>(u, off);
                else {
                    const E* q = u + row * st + c;
#pragma unroll
                    for (int e = 0; e < EPC; ++e)
                        if (c + e < Dx) {
                            if constexpr (la_f32<DT>()) r[i][e] = __float_as_uint(q[e]);
                            else r[i][e >> 1] |= (unsigned int)q[e] << (16 * (e & 1));
                        }
                }
            }
        }
    }
    __device__ __forceinline__ void store(char* t) const {
        typedef LaTile<DT, D> TT;
        char* q = t + threadIdx.x / CPR * TT::PITCH + (threadIdx.x % CPR) * EPC * (DT == 0 ? 4 : 2);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (DT == 3) {
                unsigned int h[2], m[2], l[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) v2a_split3x2(__uint_as_float(r[i][2 * e]), __uint_as_float(r[i][2 * e + 1]), h[e], m[e], l[e]);
                char* w = q + i * (NTH / CPR) * TT::PITCH;
                *(la_u32x2*)w = la_u32x2{h[0], h[1]};
                *(la_u32x2*)(w + TT::PLANE) = la_u32x2{m[0], m[1]};
                *(la_u32x2*)(w + 2 * TT::PLANE) = la_u32x2{l[0], l[1]};
            } else if constexpr (DT == 2) {
                la_u32x4 hi, lo;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float a = v2a_lo_h2<true>(r[i][e]), b = v2a_hi_h2<true>(r[i][e]);
                    hi[e] = v2a_pack_bf16x2(a, b);
                    lo[e] = v2a_pack_bf16x2(a - __uint_as_float(hi[e] << 16), b - __uint_as_float(hi[e] & 0xffff0000u));
                }
                *(la_u32x4*)(q + i * (NTH / CPR) * TT::PITCH) = hi;
                *(la_u32x4*)(q + i * (NTH / CPR) * TT::PITCH + TT::PLANE) = lo;
            } else *(la_u32x4*)(q + i * (NTH / CPR) * TT::PITCH) = r[i];
        }
    }
};

// Running log2 decays of a chunk, computed by one wave (lane = token): pair hi + lo, and the chunk's total
struct LaGate {
    float hi[LA_C], lo[LA_C];          // G_i
    float wq[LA_C], wk[LA_C];          // exp(G_i), exp(G_64 - G_i)
    float total;                       // exp(G_64)
    float pad[3];
};
// x of the lane `shr` lanes below within the 16-lane row, 0 where there is none
template <int CTRL> __device__ __forceinline__ double la_row_shr(double x) {
    const la_u32x2 u = __builtin_bit_cast(la_u32x2, x);
    return __builtin_bit_cast(double, la_u32x2{(unsigned)__builtin_amdgcn_update_dpp(0, (int)u[0], CTRL, 0xf, 0xf, true),
                                               (unsigned)__builtin_amdgcn_update_dpp(0, (int)u[1], CTRL, 0xf, 0xf, true)});
}
__device__ __forceinline__ double la_lane(double x, int l) {
    const la_u32x2 u = __builtin_bit_cast(la_u32x2, x);
    return __builtin_bit_cast(double, la_u32x2{(unsigned)__builtin_amdgcn_readlane((int)u[0], l), (unsigned)__builtin_amdgcn_readlane((int)u[1], l)});
}
// sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48 in each of them, by row swaps of the vector unit (no trip through LDS)
__device__ __forceinline__ float la_rows_sum(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// inclusive sum over the 64 lanes: inside the rows by DPP, over the rows by readlane (twelve ds_bpermute round trips otherwise: 1000 cycles)
__device__ __forceinline__ double la_running(double x, int lane) {
    x += la_row_shr<0x111>(x);
    x += la_row_shr<0x112>(x);
    x += la_row_shr<0x114>(x);
    x += la_row_shr<0x118>(x);
    const double r0 = la_lane(x, 15), r1 = la_lane(x, 31), r2 = la_lane(x, 47);
    return x + (lane < 16 ? 0.0 : lane < 32 ? r0 : lane < 48 ? r0 + r1 : r0 + r1 + r2);
}
__device__ __forceinline__ void la_gates(LaGate& s, float g, bool on, int lane) {
    const double x = la_running(on ? (double)la_clampg(g) * 1.4426950408889634 : 0.0, lane);
    const double tot = la_lane(x, 63);
    const float hi = (float)x;
    s.hi[lane] = hi;
    s.lo[lane] = (float)(x - (double)hi);
    s.wq[lane] = __builtin_amdgcn_exp2f(hi);
    s.wk[lane] = __builtin_amdgcn_exp2f((float)(tot - x));
    if (lane == 63) s.total = __builtin_amdgcn_exp2f((float)tot);
}

// The six (16-row tile, 32-slot step) units of the lower triangle of a 64 x 64 score matrix, and the wave that computes each
__device__ constexpr int la_unit_tile(int u) { return u == 0 ? 0 : u == 1 ? 1 : u < 4 ? 2 : 3; }
__device__ constexpr int la_unit_step(int u) { return u == 3 || u == 5 ? 1 : 0; }
__device__ constexpr int la_unit_wave(int u, int nw) { return nw == 1 ? 0 : nw == 2 ? u / 3 : nw == 4 ? (u < 2 ? 0 : u < 4 ? 1 : u - 2) : u; }
__device__ __forceinline__ int la_unit(int tile, int step) { return step == 0 ? (tile < 3 ? tile : 4) : tile == 2 ? 3 : 5; }
template <int DT> constexpr int la_unit_bytes() { return DT == 3 ? 64 * 48 : 64 * 32; }      // planes of 16 bytes a lane, or eight floats

template <int DT> __device__ __forceinline__ void la_put(char* p, int u, int lane, const float* x) {
    typename LaOp<DT>::C2 o;
    la_split(x, o);
    la_u32x4* q = (la_u32x4*)(p + u * la_unit_bytes<DT>()) + lane;
    if constexpr (DT == 0) {
        q[0] = la_u32x4{__float_as_uint(o.x[0]), __float_as_uint(o.x[1]), __float_as_uint(o.x[2]), __float_as_uint(o.x[3])};
        q[64] = la_u32x4{__float_as_uint(o.x[4]), __float_as_uint(o.x[5]), __float_as_uint(o.x[6]), __float_as_uint(o.x[7])};
    } else {
        q[0] = o.p[0];
        q[64] = o.p[1];
        if constexpr (DT == 3) q[128] = o.p[2];
    }
}
template <int DT> __device__ __forceinline__ void la_get(const char* p, int u, int lane, typename LaOp<DT>::C2& o) {
    const la_u32x4* q = (const la_u32x4*)(p + u * la_unit_bytes<DT>()) + lane;
    const la_u32x4 a = q[0], b = q[64];
    if constexpr (DT == 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) { o.x[e] = __uint_as_float(a[e]); o.x[4 + e] = __uint_as_float(b[e]); }
    } else {
        o.p[0] = a;
        o.p[1] = b;
        if constexpr (DT == 3) o.p[2] = q[128];
    }
}

// exp(G_i - G_j) of the four slots 4 (lane / 16) .. of the 16 tokens from t0 against the one token `one`; FIRST: the slots are i (rows), else j
template <bool SLOTS_I> __device__ __forceinline__ void la_weights(const LaGate& gt, int t0, int one, int lane, float* w) {
    const float h1 = gt.hi[one], l1 = gt.lo[one];
    const int s0 = t0 + (lane >> 4) * 4;
    const float4 h = *(const float4*)&gt.hi[s0], l = *(const float4*)&gt.lo[s0];
    const float hh[4] = {h.x, h.y, h.z, h.w}, ll[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float d = SLOTS_I ? (hh[r] - h1) + (ll[r] - l1) : (h1 - hh[r]) + (l1 - ll[r]);
        const bool in = SLOTS_I ? s0 + r >= one : s0 + r <= one;
        w[r] = in ? __builtin_amdgcn_exp2f(d) : 0.f;
    }
}

template <int DT> __device__ __forceinline__ void la_store4(typename LaT<DT>::T* p, const f32x4& x, int room, bool vec) {
    if (vec && room >= 4) {
        if constexpr (la_f32<DT>()) *(f32x4*)p = x;
        else *(la_u32x2*)p = la_u32x2{v2a_pack_h2<DT == 2>(x[0], x[1]), v2a_pack_h2<DT == 2>(x[2], x[3])};
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (r < room) p[r] = LaT<DT>::st(x[r]);
    }
}

struct LaDir {                  // one direction of the recurrence
    const float* init;          // state before the first chunk in scan order (NULL: 0)
    float* seg;                 // [B H][nseg][Dk][Dv]: local states of the segments (local) / states before them (otherwise, nseg > 1)
    float* seg_decay;           // [B H][nseg]
    int rev, vx, vy, pad;       // rev: from the last chunk to the first; v: 16-byte loads allowed
};
struct LaScan {
    LaDir dir[2];
    float* chunk;               // state before each chunk in scan order, [B H][NC][Dk][Dv] (NULL: not kept)
    // segments of two chunks (NULL: not kept): state before the second one, [B H][nseg][Dk][Dv], in the local pass without what came before the
    // segment, whose share is inner_decay [B H][nseg] of the state there; the forward direction's
    float *inner, *inner_decay;
    float* last;                // state behind the last chunk (NULL)
    void* out;
    int ndir;                   // 2: both directions, alternate workgroups
    int NC, cps, nseg, ndv, local, vq, vo, vst;
};

// One workgroup walks the chunks of one segment of one (row, head) and one tile of 16 NT NW state columns, wave w with columns 16 NT w .. of
// the state in accumulators.  OUT: the outputs as well; otherwise the states alone (of a segment that starts at 0, or before every chunk for the
// gradient).  Columns of the state never meet, so a tile of them costs k again but no exchange; scores are computed once a workgroup, by units,
// and shared through LDS.  Bound by the issue of vector, LDS and matrix instructions rather than by memory, since a chunk's stages depend on one
// another and the tiles leave room for one or two workgroups on a CU: 1 x 32768 tokens x 8 heads of 128, bf16, runs the local pass in 42 us
// (165 MB read and written, 4 TB/s, 29 % of the MFMA and 48 % of the vector issue slots taken) and OUT in 92 (303 MB, 3.3 TB/s, 26 % and 39 %);
// 8 x 2048 tokens x 8 heads 64 / 128, fp32 in planes, 36 and 77 us; 64 rows of 10 tokens x 8 heads of 48, fp32, 10 us.
// Tiles are kept twice where two workgroups still fit a CU: the waves then meet once a chunk, not before the tiles are overwritten as well
template <int DT, bool OUT> constexpr int la_scan_tiles() { return !OUT && DT == 1 ? 2 : 1; }
template <int DT, int DK, int NT, int NW, bool OUT> constexpr int la_scan_lds() {
    return (LaTile<DT, DK>::BYTES * (OUT ? 2 : 1) + LaTile<DT, 16 * NT * NW>::BYTES) * la_scan_tiles<DT, OUT>() + (OUT ? 6 * la_unit_bytes<DT>() : 0);
}
// waves per SIMD that the LDS allows, two at most: the register bound of the launch
template <int DT, int DK, int NT, int NW, bool OUT> constexpr int la_scan_waves() {
    const int n = 160 * 1024 / (la_scan_lds<DT, DK, NT, NW, OUT>() + 2304) * NW / 4;
    return n < 1 ? 1 : n > 2 ? 2 : n;
}
template <int DT, int DK, int NT, int NW, bool OUT>
__global__ __launch_bounds__(64 * NW, (la_scan_waves<DT, DK, NT, NW, OUT>())) void la_scan(LaArgs a, LaScan p) {
    typedef typename LaT<DT>::T E;
    typedef LaTile<DT, DK> TX;
    constexpr int DVT = 16 * NT * NW, NTH = 64 * NW;
    typedef LaTile<DT, DVT> TY;
    constexpr int QB = OUT ? TX::BYTES : 0;
    __shared__ __attribute__((aligned(16))) char sm[la_scan_lds<DT, DK, NT, NW, OUT>()];
    __shared__ __attribute__((aligned(16))) LaGate gts[2];
    char* sx = sm;
    char* sy = sx + TX::BYTES;
    char* sq = sy + TY::BYTES;
    char* sp = sq + QB;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int blk = blockIdx.x;
    const LaDir& m = p.dir[p.ndir == 2 ? blk & 1 : 0];
    if (p.ndir == 2) blk >>= 1;
    const int rev = m.rev;
    const int dvt = blk % p.ndv;
    blk /= p.ndv;
    const int seg = blk % p.nseg, bh = blk / p.nseg, b = bh / a.H, h = bh % a.H;
    if (!OUT && p.local && seg == p.nseg - 1 && (rev || !p.inner || seg * 2 + 1 == p.NC)) return;      // nothing follows it
    const int len = la_len(a, b), Dk = a.Dk, Dv = a.Dv, dv0 = dvt * DVT + wid * NT * 16;
    const int hq = h / (a.H / a.Hq), hk = h / (a.H / a.Hk), hv = h / (a.H / a.Hv);
    const int yroom = Dv - dvt * DVT < DVT ? Dv - dvt * DVT : DVT;
    const E* X = rev ? (const E*)a.q + b * a.qs[0] + hq * a.qs[2] : (const E*)a.k + b * a.ks[0] + hk * a.ks[2];
    const E* Y = (rev ? (const E*)a.dout + b * a.ds[0] + h * a.ds[2] : (const E*)a.v + b * a.vs[0] + hv * a.vs[2]) + dvt * DVT;
    const E* Q = (const E*)a.q + b * a.qs[0] + hq * a.qs[2];
    const long long sxt = rev ? a.qs[1] : a.ks[1], syt = rev ? a.ds[1] : a.vs[1];
    const float* g = a.g + b * a.gs[0] + h * a.gs[2];
    const long long SS = (long long)Dk * Dv;

    // This lane's state values.  OUT: S[i][n][r] is row 32 (i / 2) + 8 (lane / 16) + 4 (i % 2) + r, column c0 + 4 n (two tiles a wave: every
    // other four of 32 columns, so that a lane's outputs are eight neighbours) -- the operand of the product with q.  Else the transposed
    // tile, row 16 i + lane % 16, columns c0 + 16 n + r: four neighbours for the states that go to memory.
    f32x4 S[DK / 16][NT];
    constexpr int CS = OUT && NT == 2 ? 8 : 4, NC0 = CS == 8 ? 4 : 16;
    const int d0 = OUT ? (lane >> 4) * 8 : lane & 15, c0 = OUT ? dv0 + CS * ((lane & 15) >> 2) + (lane & 3) : dv0 + (lane >> 4) * 4;
    // OUT exchanges the state through LDS, a part of the rows at a time (in whole 32-row blocks), so that memory sees whole rows
    constexpr int NH = DK == 32 ? 1 : DK == 96 ? 3 : 2, HR = DK / NH, PER = HR * DVT / 4 / NTH;
    static_assert(!OUT || HR * DVT * 4 <= la_scan_lds<DT, DK, NT, NW, OUT>(), "the part fits");
    auto get_state = [&](const float* s0) __attribute__((always_inline)) {
        if constexpr (OUT) {
#pragma unroll
            for (int half = 0; half < NH; ++half) {
                f32x4 t[PER];
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    const int at = (e * NTH + threadIdx.x) * 4, d = half * HR + at / DVT, c = dvt * DVT + at % DVT;
                    t[e] = f32x4{0.f, 0.f, 0.f, 0.f};
                    if (d < Dk && c < Dv) {
                        const float* q = s0 + d * Dv + c;
                        if (p.vst) t[e] = *(const f32x4*)q;
                        else
#pragma unroll
                            for (int r = 0; r < 4; ++r) t[e][r] = c + r < Dv ? q[r] : 0.f;
                    }
                }
                __syncthreads();
#pragma unroll
                for (int e = 0; e < PER; ++e) ((f32x4*)sm)[e * NTH + threadIdx.x] = t[e];
                __syncthreads();
#pragma unroll
                for (int i = half * (HR / 16); i < (half + 1) * (HR / 16); ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            S[i][n][r] = ((const float*)sm)[(d0 + i / 2 * 32 + i % 2 * 4 + r - half * HR) * DVT + c0 - dvt * DVT + n * NC0];
            }
        } else
#pragma unroll
            for (int i = 0; i < DK / 16; ++i)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int d = d0 + i * 16, c = c0 + n * NC0;
                    const float* q = s0 + d * Dv + c;
                    if (d < Dk && c < Dv) {
                        if (p.vst) S[i][n] = *(const f32x4*)q;
                        else
#pragma unroll
                            for (int r = 0; r < 4; ++r) S[i][n][r] = c + r < Dv ? q[r] : 0.f;
                    }
                }
    };
    auto put_state = [&](float* dst) __attribute__((always_inline)) {
        if constexpr (OUT) {
#pragma unroll
            for (int half = 0; half < NH; ++half) {
                __syncthreads();
#pragma unroll
                for (int i = half * (HR / 16); i < (half + 1) * (HR / 16); ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            ((float*)sm)[(d0 + i / 2 * 32 + i % 2 * 4 + r - half * HR) * DVT + c0 - dvt * DVT + n * NC0] = S[i][n][r];
                __syncthreads();
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    const int at = (e * NTH + threadIdx.x) * 4, d = half * HR + at / DVT, c = dvt * DVT + at % DVT;
                    if (d < Dk && c < Dv) la_store4<0>(dst + d * Dv + c, ((const f32x4*)sm)[e * NTH + threadIdx.x], Dv - c, p.vst);
                }
            }
        } else
#pragma unroll
            for (int i = 0; i < DK / 16; ++i)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int d = d0 + i * 16, c = c0 + n * NC0;
                    if (d < Dk && c < Dv) la_store4<0>(dst + d * Dv + c, S[i][n], Dv - c, p.vst);
                }
    };
#pragma unroll
    for (int i = 0; i < DK / 16; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) S[i][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (const float* s0 = p.local ? nullptr : seg ? m.seg + ((long long)bh * p.nseg + seg) * SS : m.init ? m.init + bh * SS : nullptr) get_state(s0);
    LaLoad<DT, DK, NTH> rx, rq;
    LaLoad<DT, DVT, NTH> ry;
    float rg = 0.f;
    const int ibeg = seg * p.cps, iend = (seg + 1) * p.cps < p.NC ? (seg + 1) * p.cps : p.NC;
    // chunks with tokens: the first ones of the sequence.  The others leave the state as it is and are walked apart from the main loop, so
    // that the accumulators have one definition in it (a second path through the loop doubled their registers).
    const int nvc = (len + LA_C - 1) / LA_C, vlo = rev ? p.NC - nvc : 0, vhi = rev ? p.NC : nvc;
    const int vbeg = vlo > ibeg ? (vlo < iend ? vlo : iend) : ibeg, vend = vhi < iend ? (vhi > vbeg ? vhi : vbeg) : iend;
    auto chunk_of = [&](int i) { return rev ? p.NC - 1 - i : i; };
    auto valid = [&](int i) {
        const int n = len - chunk_of(i) * LA_C;
        return n > LA_C ? LA_C : n;
    };
    // The next chunk's rows are requested behind the score barrier: the work behind it is as long as the loads take, and their registers are
    // free before it.  Its decays are summed by the last wave meanwhile (gts[i & 1] belongs to chunk i), from values requested a chunk earlier.
    auto first = [&](int i) { return (long long)chunk_of(i) * LA_C; };
    auto fetch_x = [&](int i) { if (i < vend) rx.load(X + first(i) * sxt, sxt, valid(i), Dk, m.vx); };
    auto fetch_y = [&](int i) { if (i < vend) ry.load(Y + first(i) * syt, syt, valid(i), yroom, m.vy); };
    auto fetch_q = [&](int i) { if constexpr (OUT) if (i < vend) rq.load(Q + first(i) * a.qs[1], a.qs[1], valid(i), Dk, p.vq); };
    auto fetch_g = [&](int i) { if (wid == NW - 1 && i < vend && lane < valid(i)) rg = g[(first(i) + lane) * a.gs[1]]; };
    auto gates = [&](int i) { if (wid == NW - 1 && i < vend) la_gates(gts[i & 1], rg, lane < valid(i), lane); };
    float fac = 1.f;
    auto keep = [&](int i) __attribute__((always_inline)) {               // the state before a chunk, where it is wanted
        if (float* st = p.local ? (!rev && p.inner && i > ibeg ? p.inner + ((long long)bh * p.nseg + seg) * SS : nullptr)
                                : p.chunk && i > 0 ? p.chunk + ((long long)bh * p.NC + i) * SS : nullptr) {
            put_state(st);
            if (p.local && threadIdx.x == 0 && dvt == 0) p.inner_decay[(long long)bh * p.nseg + seg] = fac;
        }
    };
    auto skip = [&](int i) __attribute__((always_inline)) {               // a chunk without tokens
        const int c = chunk_of(i);
        if constexpr (OUT) {
            E* out = (E*)p.out + (((long long)b * a.T + (long long)c * LA_C) * a.H + h) * Dv;
            const int rows = a.T - c * LA_C < LA_C ? a.T - c * LA_C : LA_C;
            for (int r = wid * 16 + (lane & 15); r < rows; r += 16 * NW)
                for (int d = dvt * DVT + (lane >> 4) * 4; d < dvt * DVT + DVT && d < Dv; d += 16)
                    la_store4<DT>(out + (long long)r * a.H * Dv + d, f32x4{0.f, 0.f, 0.f, 0.f}, Dv - d, p.vo);
        } else keep(i);
    };
    fetch_g(vbeg);
    fetch_x(vbeg);
    fetch_y(vbeg);
    fetch_q(vbeg);
    for (int i = ibeg; i < vbeg; ++i) skip(i);
    gates(vbeg);
    fetch_g(vbeg + 1);
    for (int i = vbeg; i < vend; ++i) {
        const int c = chunk_of(i), nv = valid(i);
        if constexpr (!OUT) keep(i);
        E* out = (E*)p.out + (((long long)b * a.T + (long long)c * LA_C) * a.H + h) * Dv;
        const int rows = a.T - c * LA_C < LA_C ? a.T - c * LA_C : LA_C;
        const long long ot = (long long)a.H * Dv;
        if constexpr (la_scan_tiles<DT, OUT>() == 2) {
            sx = sm + (i & 1) * (TX::BYTES + TY::BYTES);
            sy = sx + TX::BYTES;
        } else __syncthreads();
        rx.store(sx);
        ry.store(sy);
        if constexpr (OUT) rq.store(sq);
        __syncthreads();
        const LaGate& gt = gts[i & 1];
        const bool live = i > vbeg || seg || m.init;                      // the state is not 0
        const bool keep = !OUT || i + 1 < vend || p.last;                 // somebody reads it
        const int nks = nv > 32 ? 2 : 1;
        if constexpr (OUT) {
            f32x4 O[NT][4];
#pragma unroll
            for (int u = 0; u < 6; ++u)
                if (la_unit_wave(u, NW) == wid && la_unit_tile(u) * 16 < nv) {
                    const int it = la_unit_tile(u), js = la_unit_step(u) * 32;
                    const bool two = js + 16 <= it * 16;
                    f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
                    for (int kk = 0; kk < DK / 32; ++kk) {
                        typename LaOp<DT>::In qf, kf;
                        TX::nat(sq, it * 16, kk, lane, qf);
                        TX::nat(sx, js, kk, lane, kf);
                        la_mma_in<DT>(s0, kf, qf);
                        if (two) {
                            TX::nat(sx, js + 16, kk, lane, kf);
                            la_mma_in<DT>(s1, kf, qf);
                        }
                    }
                    float w[8], x[8];
                    la_weights<false>(gt, js, it * 16 + (lane & 15), lane, w);
                    la_weights<false>(gt, js + 16, it * 16 + (lane & 15), lane, w + 4);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        x[r] = s0[r] * w[r] * a.scale;
                        x[4 + r] = s1[r] * w[4 + r] * a.scale;
                    }
                    la_put<DT>(sp, u, lane, x);
                }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int it = 0; it < 4; ++it) O[n][it] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (live) {
#pragma unroll
                for (int kk = 0; kk < DK / 32; ++kk) {
                    typename LaOp<DT>::C2 sf[NT];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float x[8];
#pragma unroll
                        for (int r = 0; r < 4; ++r) { x[r] = S[2 * kk][n][r]; x[4 + r] = S[2 * kk + 1][n][r]; }
                        la_split(x, sf[n]);
                    }
#pragma unroll
                    for (int it = 0; it < 4; ++it) {
                        typename LaOp<DT>::In qf;
                        TX::nat(sq, it * 16, kk, lane, qf);
#pragma unroll
                        for (int n = 0; n < NT; ++n) la_mma(O[n][it], sf[n], qf);
                    }
                    __builtin_amdgcn_sched_barrier(0);      // else the splits of the whole state are done at once and spill
                }
#pragma unroll
                for (int it = 0; it < 4; ++it) {
                    const float w = gt.wq[it * 16 + (lane & 15)] * a.scale;
#pragma unroll
                    for (int n = 0; n < NT; ++n) O[n][it] *= w;
                }
            }
            gates(i + 1);
            fetch_g(i + 2);
            __syncthreads();
            fetch_x(i + 1);
            fetch_y(i + 1);
            fetch_q(i + 1);
#pragma unroll 1
            for (int ks = 0; ks < nks; ++ks) {
                typename LaOp<DT>::In yf[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) TY::template tr<CS>(sy, ks, wid * NT * 16 + n * NC0, lane, yf[n]);
#pragma unroll
                for (int it = 0; it < 4; ++it)
                    if ((it >= 2 || ks == 0) && it * 16 < nv) {
                        typename LaOp<DT>::C2 pf;
                        la_get<DT>(sp, la_unit(it, ks), lane, pf);
#pragma unroll
                        for (int n = 0; n < NT; ++n) la_mma(O[n][it], yf[n], pf);
                    }
            }
            // lane: 4 NT neighbouring columns of token it * 16 + lane % 16
#pragma unroll
            for (int it = 0; it < 4; ++it) {
                const int r = it * 16 + (lane & 15), d = dv0 + (lane >> 4) * 4 * NT;
                if (r < rows && d < Dv) {
                    if (r >= nv)
#pragma unroll
                        for (int n = 0; n < NT; ++n) O[n][it] = f32x4{0.f, 0.f, 0.f, 0.f};
                    E* q = la_at<E>(out + it * 16 * ot + dv0, ((unsigned)(lane & 15) * (unsigned)ot + (unsigned)((lane >> 4) * 4 * NT)) * (unsigned)sizeof(E));
                    if constexpr (NT == 2 && !la_f32<DT>()) {
                        if (p.vo && d + 8 <= Dv) {
                            *(la_u32x4*)q = la_u32x4{v2a_pack_h2<DT == 2>(O[0][it][0], O[0][it][1]), v2a_pack_h2<DT == 2>(O[0][it][2], O[0][it][3]),
                                                     v2a_pack_h2<DT == 2>(O[1][it][0], O[1][it][1]), v2a_pack_h2<DT == 2>(O[1][it][2], O[1][it][3])};
                            continue;
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        if (d + n * 4 < Dv) la_store4<DT>(q + n * 4, O[n][it], Dv - d - n * 4, p.vo);
                }
            }
        } else {
            fetch_x(i + 1);
            fetch_y(i + 1);
            gates(i + 1);
            fetch_g(i + 2);
        }
        const float tot = gt.total;
        fac *= tot;
#pragma unroll
        for (int d = 0; d < DK / 16; ++d)
#pragma unroll
            for (int n = 0; n < NT; ++n) S[d][n] *= tot;
        const int nku = keep ? nks : 0;
#pragma unroll 1
        for (int ks = 0; ks < nku; ++ks) {
            typename LaOp<DT>::C3 yw[NT];
            const float* wsrc = (rev ? gt.wq : gt.wk) + ks * 32 + (lane >> 4) * 4;
            const float4 w0 = *(const float4*)wsrc, w1 = *(const float4*)(wsrc + 16);
            const float sc = rev ? a.scale : 1.f;
            const float w[8] = {w0.x * sc, w0.y * sc, w0.z * sc, w0.w * sc, w1.x * sc, w1.y * sc, w1.z * sc, w1.w * sc};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                typename LaOp<DT>::In yf;
                TY::template tr<CS>(sy, ks, wid * NT * 16 + n * NC0, lane, yf);
                float x[8];
                la_join(yf, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= w[e];
                la_split(x, yw[n]);
            }
#pragma unroll
            for (int d = 0; d < DK / 16; ++d) {
                typename LaOp<DT>::In xf;
                if constexpr (OUT) TX::template tr<8>(sx, ks, d / 2 * 32 + d % 2 * 4, lane, xf);
                else TX::template tr<4>(sx, ks, d * 16, lane, xf);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if constexpr (OUT) la_mma(S[d][n], xf, yw[n]);
                    else la_mma(S[d][n], yw[n], xf);
                }
                if (d & 1) __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    for (int i = vend; i < iend; ++i) skip(i);
    if (p.local) {
        put_state(m.seg + ((long long)bh * p.nseg + seg) * SS);
        if (threadIdx.x == 0 && dvt == 0) m.seg_decay[(long long)bh * p.nseg + seg] = fac;
    } else if (p.last && iend == p.NC) put_state(p.last + bh * SS);
}

// Local states of the segments -> states before them: S_0 = init, S_{s+1} = decay_s S_s + local_s, in place; W neighbours a lane, eight segments
// a round and the next round's loads ahead of this one's stores.  A chain of nseg steps a lane, bound by memory: 17 to 20 us for 8 heads of
// 128 in 64 segments (67 MB), 5.7 us for 64 heads 64 / 128 in 4.
template <int W>
__global__ __launch_bounds__(64) void la_combine(LaScan p, int nseg, long long SS) {
    typedef typename std::conditional<W == 4, f32x4, float>::type V;
    const LaDir& m = p.dir[blockIdx.z];
    const long long bh = blockIdx.y, e = ((long long)blockIdx.x * 64 + threadIdx.x) * W;
    if (e >= SS) return;
    V s = m.init ? *(const V*)(m.init + bh * SS + e) : V{};
    float* q = m.seg + bh * nseg * SS + e;
    const float* f = m.seg_decay + bh * nseg;
    // decays are loaded with the states: behind the stores, which might be to them, each would be waited for by itself
    struct Round { V x[8], z[8]; float f[8], fz[8]; } now, next;
    float* inner = blockIdx.z == 0 && p.inner ? p.inner + bh * nseg * SS + e : nullptr;
    auto get = [&](int i0, Round& r) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = i0 + j;
            r.x[j] = i + 1 < nseg ? *(const V*)(q + i * SS) : V{};
            r.f[j] = i + 1 < nseg ? f[i] : 0.f;
            if (inner) {
                const bool on = i < nseg && 2 * i + 1 < p.NC;
                r.z[j] = on ? *(const V*)(inner + i * SS) : V{};
                r.fz[j] = on ? p.inner_decay[bh * nseg + i] : 0.f;
            }
        }
    };
    get(0, now);
    for (int i0 = 0; i0 < nseg; i0 += 8) {
        get(i0 + 8, next);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i0 + j < nseg) {
                *(V*)(q + (i0 + j) * SS) = s;
                if (inner) *(V*)(inner + (i0 + j) * SS) = s * now.fz[j] + now.z[j];
                s = s * now.f[j] + now.x[j];
            }
        now = next;
    }
}

struct LaBwd {
    // state before chunk c: s_chunk[c % 2] + (b h * ns + c >> shift) Dk Dv (chunk 0: s_first)
    const float* s_chunk[2];
    int ns, shift;
    const float *s_first, *e_last;       // before the sequence / gradient of the state behind it; NULL: 0
    const float* e_seg;                  // gradient of the state behind each segment, [B H][nseg][Dk][Dv], segments from the end (the last one: e_last)
    float* e_first;                      // gradient of the state before the sequence; NULL: not wanted
    void *dq, *dk, *dv;                  // in the inputs' type, or fp32 per head where heads are shared
    float *dg, *dg_part;                 // per token, or the chunk's sum [NC][B H]
    int NC, cps, nseg, vq, vk, vv, vd, vst, fq, fk, fv;      // v: 16-byte accesses allowed; f: fp32 per-head output
};

// One workgroup walks the chunks of one segment of one (row, head) from the last to the first, with the gradient E of the state behind the
// chunk in accumulators:
//   dq_i = s (exp(G_i) S do_i + sum_j W_ij (do_i . v_j) k_j)          R_i = q_i . (the first part)
//   dk_j = exp(G_64 - G_j) E v_j + s sum_i W_ij (do_i . v_j) q_i      C_j = k_j . (the first part)
//   dv_j = exp(G_64 - G_j) E^T k_j + s sum_i W_ij (q_i . k_j) do_i
//   dg_t = exp(G_64) <S, E> + sum_{i >= t} (R_i + r_i - c_i) + sum_{j < t} C_j,   r_i = sum_{j < i} M_ij, c_j = sum_{i > j} M_ij,
//          M_ij = s W_ij (q_i . k_j)(do_i . v_j): everything whose path crosses the decay of token t,
//   E <- exp(G_64) E + s sum_i exp(G_i) q_i do_i^T.
// dg is summed from these parts, not from <q, dq> - <k, dk> over the sequence, whose difference of long sums would lose what it is after.
// Wave w owns rows 16 w .. of S, E, dq^T, dk^T and columns 16 w .. of dv^T; as dk contracts E over its columns and dv over its rows, E is
// kept twice, by rows and by columns, which costs 48 more MFMA per wave and chunk but no exchange.  Scores are computed once, by units, and
// shared through LDS; the next chunk's rows are on their way meanwhile.
// TH 2: two waves share each block of 16 rows and take half of the chunk's tokens each (E in both): where the LDS allows one workgroup of narrow
// heads on a CU, its D / 16 waves alone would leave the matrix units waiting.
// Bound by the latency of a chunk's dependent stages, with the four tiles filling the LDS of a CU (one workgroup of 128-wide heads): 4 x 4096
// tokens x 8 heads of 128, bf16, decays per token: 159 us, 284 MB read and 103 written (2.4 TB/s), 20 % of the MFMA and 37 % of the vector issue
// slots; fp32 4 x 2048 x 4 heads of 128 97 us; 8 x 2048 x 8 heads of 64 bf16 66 us, fp32 134; 8 x 2048 x 4 heads of 96 bf16 68, 80 / 96 fp32 136.  64 rows of 16 tokens x 4 heads of 64, fp32: 14 us.
template <int DT, int D> constexpr int la_bwd_halves() { return D == 32 || (D == 64 && DT != 1) ? 2 : 1; }
template <int DT, int D>
__global__ __launch_bounds__((4 * D * la_bwd_halves<DT, D>())) void la_bwd_chunks(LaArgs a, LaBwd p) {
    typedef typename LaT<DT>::T E;
    typedef LaTile<DT, D> TT;
    constexpr int TH = la_bwd_halves<DT, D>(), NB = D / 16, NW = NB * TH, NTH = 64 * NW, KK = D / 32, TPW = 4 / TH;
    constexpr bool AHEAD = DT != 0 || D < 128;      // fp32 rows of 128: their registers would spill
    constexpr int UB = 6 * la_unit_bytes<DT>();
    constexpr int NBUF = 4 * TT::BYTES + 3 * UB + 10240 <= 160 * 1024 ? 3 : 1;      // score buffers: all three at once where they fit
    __shared__ __attribute__((aligned(16))) char sm[4 * TT::BYTES + NBUF * UB];
    __shared__ __attribute__((aligned(16))) LaGate gts[2];
    __shared__ float sr[NB][LA_C], sc[NB][LA_C], rm[4][LA_C], cm[2][LA_C], sz[NB];
    char *sq = sm, *sk = sq + TT::BYTES, *sv = sk + TT::BYTES, *sd = sv + TT::BYTES, *s1 = sd + TT::BYTES;
    char *s2 = s1 + (NBUF == 3 ? UB : 0), *s3 = s2 + (NBUF == 3 ? UB : 0);
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, l4 = (lane >> 4) * 4, blk = TH == 1 ? wid : wid % NB, t0 = TH == 1 ? 0 : wid / NB * TPW;      // rows 16 blk .., token tiles t0 ..
    const int seg = blockIdx.x % p.nseg, bh = blockIdx.x / p.nseg, b = bh / a.H, h = bh % a.H;
    const int Dk = a.Dk, Dv = a.Dv, w0 = blk * 16;
    const int hq = h / (a.H / a.Hq), hk = h / (a.H / a.Hk), hv = h / (a.H / a.Hv);
    const long long SS = (long long)Dk * Dv;
    const int len = la_len(a, b);
    const E* Q = (const E*)a.q + b * a.qs[0] + hq * a.qs[2];
    const E* K = (const E*)a.k + b * a.ks[0] + hk * a.ks[2];
    const E* V = (const E*)a.v + b * a.vs[0] + hv * a.vs[2];
    const E* G = (const E*)a.dout + b * a.ds[0] + h * a.ds[2];
    const float* g = a.g + b * a.gs[0] + h * a.gs[2];

    // four values of each of the rows l16 of this wave's token tiles of a gradient: shared heads keep fp32 per head (rows of H heads), others their own type
    auto put = [&](void* base, int f32, int Hx, int hx, int Dx, int c, const f32x4 (&x)[TPW]) __attribute__((always_inline)) {
        const int left = la_here(a.T - c * LA_C), room = Dx - w0 - l4, ld = la_here((f32 ? a.H : Hx) * Dx);
        const long long at = ((long long)b * a.T + (long long)c * LA_C) * ld + (f32 ? h : hx) * Dx + w0;
        const unsigned off = (unsigned)l16 * (unsigned)ld + (unsigned)l4;
        if (room <= 0) return;
        auto rows = [&](auto&& one) __attribute__((always_inline)) {
#pragma unroll
            for (int tt = 0; tt < TPW; ++tt)
                if ((t0 + tt) * 16 + l16 < left) one(at + (long long)((t0 + tt) * 16) * ld, x[tt]);
        };
        if (Dx % 4 == 0) {
            if (f32) rows([&](long long o, const f32x4& y) { *la_at<f32x4>((float*)base + o, off * 4u) = y; });
            else rows([&](long long o, const f32x4& y) { la_store4<DT>(la_at<E>((E*)base + o, off * (unsigned)sizeof(E)), y, 4, true); });
        } else {
            if (f32) rows([&](long long o, const f32x4& y) { la_store4<0>(la_at<float>((float*)base + o, off * 4u), y, room, false); });
            else rows([&](long long o, const f32x4& y) { la_store4<DT>(la_at<E>((E*)base + o, off * (unsigned)sizeof(E)), y, room, false); });
        }
    };
    // this segment's chunks chi, chi - 1, .. clo; those from nvc on have no tokens
    const int chi = p.NC - 1 - seg * p.cps, clo = chi - p.cps + 1 > 0 ? chi - p.cps + 1 : 0;
    const int nvc = (len + LA_C - 1) / LA_C, cfirst = chi < nvc ? chi : nvc - 1;
    for (int c = chi; c > cfirst && c >= clo; --c) {
        const f32x4 z[TPW] = {};
        put(p.dq, p.fq, a.Hq, hq, Dk, c, z);
        put(p.dk, p.fk, a.Hk, hk, Dk, c, z);
        put(p.dv, p.fv, a.Hv, hv, Dv, c, z);
        if (wid == 0 && p.dg && c * LA_C + lane < a.T) p.dg[((long long)b * a.T + (long long)c * LA_C + lane) * a.H + h] = 0.f;
        if (threadIdx.x == 0 && p.dg_part) p.dg_part[(long long)c * a.B * a.H + bh] = 0.f;
    }

    // E by rows: e1[kk][half][r] is row w0 + l16, column 32 kk + 8 (lane / 16) + 4 half + r; by columns: e2, row and column exchanged
    f32x4 e1[KK][2], e2[KK][2];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int half = 0; half < 2; ++half) e1[kk][half] = e2[kk][half] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto state_rows = [&](const float* st, f32x4 (&x)[KK][2]) __attribute__((always_inline)) {      // zeros where there is no value
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int d = kk * 32 + l4 * 2 + half * 4;
                x[kk][half] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (st && w0 + l16 < Dk && d < Dv) {
                    const float* q = la_at<float>(st, (unsigned)((w0 + l16) * Dv + l4 * 2) * 4u) + kk * 32 + half * 4;
                    if (p.vst) x[kk][half] = *(const f32x4*)q;
                    else
#pragma unroll
                        for (int r = 0; r < 4; ++r) x[kk][half][r] = d + r < Dv ? q[r] : 0.f;
                }
            }
    };
    const float* ep = seg ? p.e_seg + ((long long)bh * p.nseg + seg) * SS : p.e_last ? p.e_last + bh * SS : nullptr;
    bool have_e = ep != nullptr;
    if (ep) {
        state_rows(ep, e1);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = kk * 32 + l4 * 2 + half * 4 + r, c = w0 + l16;
                    const float x = ep[(d < Dk ? d : 0) * Dv + (c < Dv ? c : 0)];
                    e2[kk][half][r] = d < Dk && c < Dv ? x : 0.f;
                }
    }
    LaLoad<DT, D, NTH> rq, rk, rv, rd;
    float rgn = 0.f;      // the next chunk's decays, in the last wave
    auto valid = [&](int c) { return len - c * LA_C < LA_C ? len - c * LA_C : LA_C; };
    auto fetch = [&](int c) __attribute__((always_inline)) {
        if (c < clo) return;
        const long long f0 = (long long)c * LA_C;
        const int nv = valid(c);
        rq.load(Q + f0 * a.qs[1], a.qs[1], nv, Dk, p.vq);
        rk.load(K + f0 * a.ks[1], a.ks[1], nv, Dk, p.vk);
        rv.load(V + f0 * a.vs[1], a.vs[1], nv, Dv, p.vv);
        rd.load(G + f0 * a.ds[1], a.ds[1], nv, Dv, p.vd);
    };
    auto fetch_g = [&](int c) { if (wid == NW - 1 && c >= clo && lane < valid(c)) rgn = g[((long long)c * LA_C + lane) * a.gs[1]]; };
    auto gates = [&](int c) { if (wid == NW - 1 && c >= clo) la_gates(gts[c & 1], rgn, lane < valid(c), lane); };
    auto state_of = [&](int c) { return c == 0 ? (p.s_first ? p.s_first + bh * SS : nullptr) : p.s_chunk[c & 1] + ((long long)bh * p.ns + (c >> p.shift)) * SS; };
    f32x4 xs[KK][2];
    if (cfirst >= clo) {
        fetch_g(cfirst);
        fetch(cfirst);
        state_rows(state_of(cfirst), xs);
        gates(cfirst);
        fetch_g(cfirst - 1);
    }
    f32x4 acc[TPW];
    float raw[3][8];
    // d decay of a chunk (first wave, lane = token): its parts are gathered from LDS while the next chunk's rows are stored, and summed up later
    double up = 0.0, down = 0.0, cross = 0.0;
    bool gone = false;
    auto gather = [&](int c) __attribute__((always_inline)) {
        const int nv = valid(c);
        const LaGate& gt = gts[c & 1];
        float u = 0.f, dn = 0.f, z = 0.f;
#pragma unroll
        for (int w = 0; w < NB; ++w) {
            u += sr[w][lane];
            dn += sc[w][lane];
            z += sz[w];
        }
        // parts that no unit of the lower triangle wrote are left out
        float r = 0.f, m = 0.f;
#pragma unroll
        for (int jt = 0; jt < 4; ++jt)
            if (lane >= jt * 16) r += rm[jt][lane];
        if (lane < 32) m += cm[0][lane];
        if (nv > 32) m += cm[1][lane];
        const float g2 = lane ? (gt.hi[lane] - gt.hi[lane - 1]) + (gt.lo[lane] - gt.lo[lane - 1]) : gt.hi[0];
        gone = __builtin_amdgcn_exp2f(g2) == 0.f || lane >= nv;
        up = lane < nv ? ((double)u + (double)r) - (double)m : 0.0;
        down = lane < nv ? (double)dn : 0.0;
        cross = (double)z * (double)gt.total;
    };
    auto decays = [&](int c) __attribute__((always_inline)) {
        const double to = la_running(down, lane) - down, all = la_running(up, lane), from = la_lane(all, 63) - all + up;
        double d = gone ? 0.0 : cross + from + to;
        const long long t = (long long)c * LA_C + lane;
        if (p.dg && t < a.T) p.dg[((long long)b * a.T + t) * a.H + h] = (float)d;
        if (p.dg_part) {
            d = wave_sum_d(d);
            if (lane == 0) p.dg_part[(long long)c * a.B * a.H + bh] = (float)d;
        }
    };
    for (int c = cfirst; c >= clo; --c) {
        const int nv = valid(c);
        const LaGate& gt = gts[c & 1];
        if (!AHEAD && c < cfirst) fetch(c);
        __syncthreads();
        rq.store(sq);
        rk.store(sk);
        rv.store(sv);
        rd.store(sd);
        if (wid == 0 && c < cfirst) gather(c + 1);
        __syncthreads();
        {
            float z = 0.f;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int r = 0; r < 4; ++r) z += xs[kk][half][r] * e1[kk][half][r];
            z = wave_sum(z);
            if (lane == 0 && t0 == 0) sz[blk] = z;
        }
        // W (do . v) with lane = i, slots = j: the operand of dq
        auto unit1 = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < 6; ++u) {
                const int it = la_unit_tile(u), js = la_unit_step(u) * 32;
                if ((NBUF == 3 && NW == 8 ? 6 + u / 3 : la_unit_wave(u, NW)) != wid || it * 16 >= nv) continue;
                f32x4 c0 = {0.f, 0.f, 0.f, 0.f}, c1 = {0.f, 0.f, 0.f, 0.f};
                const bool two = js + 16 <= it * 16;
                for (int kk = 0; kk * 32 < Dv; ++kk) {
                    typename LaOp<DT>::In df, vf;
                    TT::nat(sd, it * 16, kk, lane, df);
                    TT::nat(sv, js, kk, lane, vf);
                    la_mma_in<DT>(c0, vf, df);
                    if (two) {
                        TT::nat(sv, js + 16, kk, lane, vf);
                        la_mma_in<DT>(c1, vf, df);
                    }
                }
                float w[8], x[8];
                la_weights<false>(gt, js, it * 16 + l16, lane, w);
                la_weights<false>(gt, js + 16, it * 16 + l16, lane, w + 4);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = c0[r] * w[r] * a.scale;
                    x[4 + r] = c1[r] * w[4 + r] * a.scale;
                }
                la_put<DT>(s1, u, lane, x);
            }
        };
        // W (x . y) with lane = j, slots = i: the operands of dk (x = do, y = v) and dv (x = q, y = k); unit u is tile 3 - tile(u), step 1 - step(u)
        auto unit23 = [&](const char* sx, const char* sy, char* dst, int Dx, bool third) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < 6; ++u) {
                const int jt = 3 - la_unit_tile(u), is = 32 - la_unit_step(u) * 32;
                constexpr int per = NW >= 6 ? 1 : NW == 4 ? 2 : 3;
                const int at = u % per;
                if (la_unit_wave(u, NW) != wid || jt * 16 >= nv || is >= nv) continue;
                f32x4 c0 = {0.f, 0.f, 0.f, 0.f}, c1 = {0.f, 0.f, 0.f, 0.f};
                const bool first = is + 16 > jt * 16;
                for (int kk = 0; kk * 32 < Dx; ++kk) {
                    typename LaOp<DT>::In xf, yf;
                    TT::nat(sy, jt * 16, kk, lane, yf);
                    if (first) {
                        TT::nat(sx, is, kk, lane, xf);
                        la_mma_in<DT>(c0, xf, yf);
                    }
                    TT::nat(sx, is + 16, kk, lane, xf);
                    la_mma_in<DT>(c1, xf, yf);
                }
                float w[8], x[8];
                const int j = jt * 16 + l16;
                la_weights<true>(gt, is, j, lane, w);
                la_weights<true>(gt, is + 16, j, lane, w + 4);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = c0[r] * w[r] * a.scale;
                    x[4 + r] = c1[r] * w[4 + r] * a.scale;
                }
                la_put<DT>(dst, u, lane, x);
                if (!third) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) { raw[at][r] = c0[r]; raw[at][4 + r] = c1[r]; }
                } else {
                    float col = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int i = is + (e < 4 ? e : 12 + e) + l4;
                        float m = i > j ? x[e] * raw[at][e] : 0.f;
                        col += m;
                        m += v2a_dpp<0xB1>(m);              // sum over the 16 lanes of a row group
                        m += v2a_dpp<0x4E>(m);
                        m += v2a_dpp<0x141>(m);
                        m += v2a_dpp<0x140>(m);
                        if (l16 == 0) rm[jt][i] = m;
                    }
                    col = la_rows_sum(col);
                    if (lane < 16) cm[is >> 5][j] = col;
                }
            }
        };
        auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < TPW; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        };
        // a state's rows (or columns) times the tokens' rows in `t`, weighted by w.  `form` is the state's: three planes (exact fp32) for
        // dq and dk, whose products with q and k make the fp32 d decay, two for dv
        auto through = [&](const f32x4 (&x)[KK][2], const char* t, const float* w, float mul, auto form) __attribute__((always_inline)) {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                float y[8];
#pragma unroll
                for (int r = 0; r < 4; ++r) { y[r] = x[kk][0][r]; y[4 + r] = x[kk][1][r]; }
                decltype(form) sf;
                la_split(y, sf);
#pragma unroll
                for (int tt = 0; tt < TPW; ++tt) {
                    typename LaOp<DT>::In tf;
                    TT::nat(t, (t0 + tt) * 16, kk, lane, tf);
                    la_mma(acc[tt], sf, tf);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int tt = 0; tt < TPW; ++tt) acc[tt] *= w[(t0 + tt) * 16 + l16] * mul;
        };
        // and its product with the tokens' own rows: this wave's share
        auto with_own = [&](const char* own, float* dst) __attribute__((always_inline)) {
#pragma unroll
            for (int tt = 0; tt < TPW; ++tt) {
                float y[4];
                TT::four(own, (t0 + tt) * 16 + l16, w0 + l4, y);
                const float s = la_rows_sum((acc[tt][0] * y[0] + acc[tt][1] * y[1]) + (acc[tt][2] * y[2] + acc[tt][3] * y[3]));
                if (lane < 16) dst[(t0 + tt) * 16 + lane] = s;
            }
        };
        // the part within the chunk: columns w0 .. of the tokens in `t` times the shared scores
        auto within = [&](const char* t, const char* units, bool mirrored) __attribute__((always_inline)) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
                if (ks * 32 < nv) {
                    typename LaOp<DT>::In tf;
                    TT::template tr<4>(t, ks, w0, lane, tf);
#pragma unroll
                    for (int u = 0; u < 6; ++u) {
                        const int tile = mirrored ? 3 - la_unit_tile(u) : la_unit_tile(u);
                        if ((mirrored ? 1 - la_unit_step(u) : la_unit_step(u)) != ks || tile * 16 >= nv) continue;
                        if (TH == 2 && tile / TPW * TPW != t0) continue;
                        typename LaOp<DT>::C2 xf;
                        la_get<DT>(units, u, lane, xf);
                        la_mma(acc[tile % TPW], tf, xf);
                    }
                }
        };
        auto emit = [&](void* base, int f32, int Hx, int hx, int Dx) __attribute__((always_inline)) {
#pragma unroll
            for (int tt = 0; tt < TPW; ++tt) {
                if ((t0 + tt) * 16 + l16 >= nv) acc[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            put(base, f32, Hx, hx, Dx, c, acc);
        };
        const float* sp = state_of(c);
        if (wid == 0 && c < cfirst) decays(c + 1);
        unit1();
        if constexpr (NBUF == 3) {
            unit23(sd, sv, s2, Dv, false);
            unit23(sq, sk, s3, Dk, true);
        }
        __syncthreads();
        clear();
        if (AHEAD) fetch(c - 1);
        if (sp && w0 < Dk) through(xs, sd, gt.wq, a.scale, typename LaOp<DT>::C3());
        with_own(sq, sr[blk]);
        LA_FENCE;
        within(sk, s1, false);
        LA_FENCE;
        emit(p.dq, p.fq, a.Hq, hq, Dk);
        LA_FENCE;
        if (c > clo) state_rows(state_of(c - 1), xs);
        gates(c - 1);
        fetch_g(c - 2);
        if constexpr (NBUF == 1) {
            __syncthreads();
            unit23(sd, sv, s2, Dv, false);
            __syncthreads();
        }
        clear();
        if (have_e && w0 < Dk) through(e1, sv, gt.wk, 1.f, typename LaOp<DT>::C3());
        with_own(sk, sc[blk]);
        LA_FENCE;
        within(sq, s2, true);
        LA_FENCE;
        emit(p.dk, p.fk, a.Hk, hk, Dk);
        LA_FENCE;
        if constexpr (NBUF == 1) {
            __syncthreads();
            unit23(sq, sk, s3, Dk, true);
            __syncthreads();
        }
        clear();
        if (have_e && w0 < Dv) through(e2, sk, gt.wk, 1.f, typename LaOp<DT>::C2());
        within(sd, s3, true);
        LA_FENCE;
        emit(p.dv, p.fv, a.Hv, hv, Dv);
        LA_FENCE;
        // E of the chunk before, if anybody reads it (a loop of no rounds, not a branch: the accumulators keep one definition)
        const int nks = c > clo || p.e_first ? (nv > 32 ? 2 : 1) : 0;
        have_e = true;
        const float tot = gt.total;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                e1[kk][half] *= tot;
                e2[kk][half] *= tot;
            }
#pragma unroll 1
        for (int ks = 0; ks < nks; ++ks) {
            const float* wsrc = gt.wq + ks * 32 + l4;
            const float4 wa = *(const float4*)wsrc, wb = *(const float4*)(wsrc + 16);
            const float w[8] = {wa.x * a.scale, wa.y * a.scale, wa.z * a.scale, wa.w * a.scale,
                                wb.x * a.scale, wb.y * a.scale, wb.z * a.scale, wb.w * a.scale};
            auto weighted = [&](const typename LaOp<DT>::In& f, typename LaOp<DT>::C3& o) __attribute__((always_inline)) {
                float x[8];
                la_join(f, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= w[e];
                la_split(x, o);
            };
            typename LaOp<DT>::In qf, df;
            typename LaOp<DT>::C3 qw, dw;
            TT::template tr<4>(sq, ks, w0, lane, qf);
            TT::template tr<4>(sd, ks, w0, lane, df);
            weighted(qf, qw);
            weighted(df, dw);
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    TT::template tr<8>(sd, ks, kk * 32 + half * 4, lane, df);
                    la_mma(e1[kk][half], df, qw);
                    TT::template tr<8>(sq, ks, kk * 32 + half * 4, lane, qf);
                    la_mma(e2[kk][half], qf, dw);
                }
        }
    }
    __syncthreads();
    if (wid == 0 && cfirst >= clo) {
        gather(clo);
        decays(clo);
    }
    if (p.e_first && clo == 0 && t0 == 0 && w0 + l16 < Dk)
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int d = kk * 32 + l4 * 2 + half * 4;
                if (d < Dv) la_store4<0>(p.e_first + bh * SS + (w0 + l16) * Dv + d, e1[kk][half], Dv - d, p.vst);
            }
}

// gradients of shared heads: the heads of a group summed in order, rounded once (5 x 777 tokens, 6 heads of 40 to 2, q and k: 4.7 us, mostly the launch)
struct LaShare { const float* src; void* dst; int Hx, rep, D; };
struct LaShares { LaShare of[3]; };      // q, k, v; src NULL: not shared
template <int DT>
__global__ __launch_bounds__(256) void la_share(LaShares all, long long rows) {
    typedef typename LaT<DT>::T E;
    const LaShare m = all.of[blockIdx.y];
    if (!m.src) return;
    E* dst = (E*)m.dst;
    const long long n = rows * m.Hx * m.D;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        const long long r = i / m.D;
        const int c = (int)(i - r * m.D);
        float s = 0.f;
        for (int j = 0; j < m.rep; ++j) s += m.src[(r * m.rep + j) * m.D + c];
        dst[i] = LaT<DT>::st(s);
    }
}

// d decay of a per-head decay: the sum over all chunks and rows, one workgroup per head, in fp64 (64 rows x 1 chunk: 3 us, the launch)
__global__ __launch_bounds__(256) void la_dg_heads(const float* dgt, float* dg, long long rows, int H) {
    __shared__ double red[4];
    double s = 0.0;
    for (long long r = threadIdx.x; r < rows; r += 256) s += dgt[r * H + blockIdx.x];
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) dg[blockIdx.x] = (float)((red[0] + red[1]) + (red[2] + red[3]));
}

// ---------------------------------------------------------------------------------------------------------------------- single tokens
// One workgroup per (row, head): reads and writes the Dk x Dv state once, which is all of the traffic that counts.  lv lanes of 16 bytes cover
// a state row, the other lanes take further rows, eight of them under way per lane.  Rows that name the same slot are taken by the first of
// them, in row order, as successive tokens.  Bound by memory: 512 rows x 16 heads of 128 x 128 take 230 us, 4.7 of the 5.1 TB/s that a copy of
// that size reaches; one row of 8 heads of 48 x 48 takes 4.9 us, an empty launch 3.7.  Streaming (nontemporal) accesses: 231 us against 247.
template <int DT, int W>
__global__ __launch_bounds__(256) void la_step_kernel(const void* q_, const void* k_, const void* v_, const float* g, float* state, const int* slots,
                                                      void* out_, long long qb_, long long qh_, long long kb_, long long kh_, long long vb_, long long vh_,
                                                      long long gb_, long long gh_, int B, int N, int H, int Hq, int Hk, int Hv, int Dk, int Dv, int lv, float scale) {
    typedef typename LaT<DT>::T E;
    constexpr int AHEAD = 8;
    __shared__ float qs[LA_DMAX], ks[LA_DMAX];
    __shared__ float red[4][LA_DMAX];
    __shared__ int nexts[256];
    const int x = threadIdx.x, h = blockIdx.x % H;
    int b = blockIdx.x / H, slot = b;
    E* out = (E*)out_;
    bool more = false;
    if (slots) {
        slot = slots[b];
        int low = 0, high = 0;
        for (int j = x; j < B; j += 256) {
            const bool same = slots[j] == slot;
            low |= same && j < b;
            high |= same && j > b;
        }
        if (slot < 0 || slot >= N) {
            if (x < Dv) out[((long long)b * H + h) * Dv + x] = LaT<DT>::st(0.f);
            return;
        }
        if (__syncthreads_or(low)) return;
        more = __syncthreads_or(high);
    }
    float* S = state + ((long long)slot * H + h) * Dk * Dv;
    const int c = (x & (lv - 1)) * W, r0 = x / lv, rg = 256 / lv, lane = x & 63;
    for (;;) {
        const E* q = (const E*)q_ + b * qb_ + (h / (H / Hq)) * qh_;
        const E* k = (const E*)k_ + b * kb_ + (h / (H / Hk)) * kh_;
        const E* v = (const E*)v_ + b * vb_ + (h / (H / Hv)) * vh_;
        const float w = __builtin_amdgcn_exp2f(la_clampg(g[b * gb_ + h * gh_]) * 1.44269504088896340736f);
        if (x < Dk) { qs[x] = LaT<DT>::ld(q[x]) * scale; ks[x] = LaT<DT>::ld(k[x]); }
        float vv[W], o[W];
#pragma unroll
        for (int i = 0; i < W; ++i) { vv[i] = c + i < Dv ? LaT<DT>::ld(v[c + i]) : 0.f; o[i] = 0.f; }
        __syncthreads();
        for (int r1 = r0; r1 < Dk; r1 += AHEAD * rg) {
            float y[AHEAD][W];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int r = r1 + j * rg;
                if (r < Dk && c < Dv) {
                    if constexpr (W == 4) *(f32x4*)y[j] = __builtin_nontemporal_load((const f32x4*)(S + r * Dv + c));
                    else y[j][0] = S[r * Dv + c];
                }
            }
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int r = r1 + j * rg;
                if (r < Dk && c < Dv) {
                    const float kr = ks[r], qr = qs[r];
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        y[j][i] = y[j][i] * w + kr * vv[i];
                        o[i] += qr * y[j][i];
                    }
                    if constexpr (W == 4) __builtin_nontemporal_store(*(const f32x4*)y[j], (f32x4*)(S + r * Dv + c));
                    else S[r * Dv + c] = y[j][0];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < W; ++i)
            for (int m = lv; m < 64; m *= 2) o[i] += __shfl_xor(o[i], m, 64);
        // one sum a wave, or one a pair of waves where 128 lanes share a row
        const int groups = lv > 64 ? 2 : 4, mine = lv > 64 ? x >> 7 : x >> 6;
        if ((lane < lv || lv > 64) && c < Dv)
#pragma unroll
            for (int i = 0; i < W; ++i) red[mine][c + i] = o[i];
        __syncthreads();
        if (x < Dv) out[((long long)b * H + h) * Dv + x] = LaT<DT>::st(groups == 2 ? red[0][x] + red[1][x] : (red[0][x] + red[1][x]) + (red[2][x] + red[3][x]));
        if (!more) return;
        int next = 0x7fffffff;
        for (int j = b + 1 + x; j < B; j += 256)
            if (slots[j] == slot) { next = j; break; }
        nexts[x] = next;
        __syncthreads();
        for (int j = 0; j < 256; ++j) next = min(next, nexts[j]);
        if (next == 0x7fffffff) return;
        b = next;
        __syncthreads();
    }
}

bool la_dims(int B, int T, int H, int Hq, int Hk, int Hv, int Dk, int Dv, int dtype) {
    return B >= 0 && T >= 0 && H > 0 && Hq > 0 && Hk > 0 && Hv > 0 && H % Hq == 0 && H % Hk == 0 && H % Hv == 0 && Dk > 0 && Dk <= LA_DMAX && Dv > 0 &&
           Dv <= LA_DMAX && dtype >= 0 && dtype <= 2 && (long long)B * H * (T / 64 + 1) < (1ll << 23) &&      // grid x block stays below 2^32 threads,
           (long long)H * LA_DMAX < (1ll << 24);                                                      // 16 rows of all heads below 2^31 bytes
}

LaArgs la_args(const void* q, const void* k, const void* v, const float* g, const float* state, const int32_t* lens, const void* dout, const int64_t* st, int B,
               int T, int H, int Hq, int Hk, int Hv, int Dk, int Dv, float scale) {
    LaArgs a{};
    a.q = q; a.k = k; a.v = v; a.g = g; a.state = state; a.lens = lens; a.dout = dout;
    for (int i = 0; i < 3; ++i) { a.qs[i] = st[i]; a.ks[i] = st[3 + i]; a.vs[i] = st[6 + i]; a.gs[i] = st[9 + i]; a.ds[i] = dout ? st[12 + i] : 0; }
    a.B = B; a.T = T; a.H = H; a.Hq = Hq; a.Hk = Hk; a.Hv = Hv; a.Dk = Dk; a.Dv = Dv; a.scale = scale;
    return a;
}

size_t la_up(size_t n) { return (n + 255) & ~(size_t)255; }

#define LA_BY_TYPE(dtype, CALL)      \
    do {                             \
        if ((dtype) == 0) { CALL(0); } \
        else if ((dtype) == 1) { CALL(1); } \
        else { CALL(2); }            \
    } while (0)

// How a call is cut: columns of the state per workgroup (dvt) and segments of the sequence.  One workgroup per CU and more keep the chip busy;
// where (row, head) pairs and column tiles are fewer, the chunks are cut into segments of at least `least`, whose states come from a first pass.
struct LaPlan {
    int dvt, ndv, NC, cps, nseg;
};
// State columns per workgroup; both widths from 65 to 96: tiles of 96 and six waves
int la_dvt(int Dk, int Dv, int dtype) {
    return Dv <= 32 ? 32 : Dk > 64 && Dk <= 96 && Dv > 64 && Dv <= 96 ? 96 : Dv <= 64 || (dtype == 0 && Dk > 64) ? 64 : 128;
}
// `wg` workgroups without segments, `room` for as many at once; a chunk costs `more` tenths with segments of what it costs without (the pass for
// their states), and a segment about one chunk of its own.  One or two rounds of the chip, whichever ends first: a round that is nearly empty takes
// as long as a full one.
LaPlan la_plan(int T, int Dk, int Dv, int dtype, long wg, int room, int more) {
    constexpr int least = 2;
    LaPlan p;
    p.dvt = la_dvt(Dk, Dv, dtype);
    p.ndv = cdiv(Dv, p.dvt);
    p.NC = cdiv(T, LA_C);
    p.nseg = 1;
    p.cps = p.NC;
    long best = 10l * p.NC;
    if (p.NC >= 2 * least && wg > 0 && wg < room)
        for (int k = 1; k <= 2; ++k) {
            int cps = cdiv(p.NC, (int)(k * room / wg));
            if (cps < least) cps = least;
            const int nseg = cdiv(p.NC, cps);
            const long cost = (long)more * cdiv(nseg * wg, room) * (cps + 1);
            if (nseg > 1 && cost < best) { best = cost; p.cps = cps; p.nseg = nseg; }
        }
    return p;
}
// as many workgroups as fit the chip at once, by their LDS: two on a CU where they take 80 KB at most, else one.  More segments than that only
// add states: 8 x 2048 tokens x 8 heads 64 / 128 fp32 takes 119 us with 256 workgroups, 132 with 512, 158 with 1024; 1 x 32768 x 8 heads of 128 bf16
// 181, 158, 193 (sums of the three kernels)
LaPlan la_plan_fwd(int BH, int T, int Dk, int Dv, int dtype) {
    return la_plan(T, Dk, Dv, dtype, (long)BH * cdiv(Dv, la_dvt(Dk, Dv, dtype)), dtype == 1 || (Dk <= 64 && Dv <= 64) ? 512 : 256, 15);
}
// by the gradient kernel, whose workgroups have all columns
LaPlan la_plan_bwd(int BH, int T, int Dk, int Dv, int dtype) {
    return la_plan(T, Dk, Dv, dtype, BH, (Dk <= 32 && Dv <= 32) || (dtype == 1 && Dk <= 64 && Dv <= 64) ? 512 : 256, 12);
}

int la_vec(const void* p, const long long* st, int B, int T, int H, int D, int dtype) {
    const long long es = dtype == 0 ? 4 : 2;
    if (((uintptr_t)p & 15) || D * es % 16) return 0;
    if (T > 1 && (st[1] < 0 || st[1] * es * LA_C > 0x7fffffffll)) return 0;      // rows of a chunk within 32-bit offsets
    return !((B > 1 && st[0] * es % 16) || (T > 1 && st[1] * es % 16) || (H > 1 && st[2] * es % 16));
}

// fp32 by the fp32 MFMA: where its tiles leave room for two workgroups on a CU and three planes of them do not (64 x 10 tokens x 8 heads of 48:
// 10.6 us against 15.3; 8 x 2048 tokens x 8 heads 64 / 128, which do not fit twice either way: 100 us against 75)
bool la_plain_fp32(int Dk, int dvt) { return Dk <= 64 && dvt <= 64; }

template <int DT, int DK, bool OUT> int la_scan_dv(const LaArgs& a, const LaScan& p, int dvt, hipStream_t s) {
    const dim3 grid((unsigned)((long long)a.B * a.H * p.ndv * p.nseg * p.ndir));
    if constexpr (!(DT == 3 && DK < 128)) {
        if (dvt == 32) hipLaunchKernelGGL((la_scan<DT, DK, 1, 2, OUT>), grid, dim3(128), 0, s, a, p);
        else if (dvt == 64) hipLaunchKernelGGL((la_scan<DT, DK, 1, 4, OUT>), grid, dim3(256), 0, s, a, p);
    }
    if constexpr (DT != 0 && !(DT == 3 && DK == 128)) {      // fp32: planes of 128 columns, and of 64 beside keys over 64 wide (all three tiles: 157 KB)
        if (dvt == 128) {
            if constexpr (DK == 32 || (OUT && DT == 1)) hipLaunchKernelGGL((la_scan<DT, DK, 2, 4, OUT>), grid, dim3(256), 0, s, a, p);
            else hipLaunchKernelGGL((la_scan<DT, DK, 1, 8, OUT>), grid, dim3(512), 0, s, a, p);
        }
    }
    V2A_CHECK_LAUNCH();
    return V2A_OK;
}
template <int DT, bool OUT> int la_scan_dk(const LaArgs& a, const LaScan& p, int dvt, hipStream_t s) {
    if (a.Dk <= 32) return la_scan_dv<DT, 32, OUT>(a, p, dvt, s);
    if (a.Dk <= 64) return la_scan_dv<DT, 64, OUT>(a, p, dvt, s);
    if constexpr (DT != 0)
        if (dvt == 96) {
            hipLaunchKernelGGL((la_scan<DT, 96, 1, 6, OUT>), dim3((unsigned)((long long)a.B * a.H * p.nseg * p.ndir)), dim3(384), 0, s, a, p);
            V2A_CHECK_LAUNCH();
            return V2A_OK;
        }
    if constexpr (DT == 0) return V2A_ERR_ARG;      // la_plain_fp32
    else return la_scan_dv<DT, 128, OUT>(a, p, dvt, s);
}
template <bool OUT> int la_launch_scan(const LaArgs& a, const LaScan& p, int dvt, int dtype, hipStream_t s) {
    if (dtype == 0) return la_plain_fp32(a.Dk, dvt) ? la_scan_dk<0, OUT>(a, p, dvt, s) : la_scan_dk<3, OUT>(a, p, dvt, s);
    return dtype == 1 ? la_scan_dk<1, OUT>(a, p, dvt, s) : la_scan_dk<2, OUT>(a, p, dvt, s);
}

// States before the segments: local ones, then their combination
int la_segments(const LaArgs& a, LaScan p, const LaPlan& pl, int dtype, hipStream_t s) {
    p.vst = a.Dv % 4 == 0;
    p.NC = pl.NC; p.cps = pl.cps; p.nseg = pl.nseg; p.ndv = pl.ndv;
    p.local = 1; p.chunk = nullptr; p.last = nullptr;
    const int rc = la_launch_scan<false>(a, p, pl.dvt, dtype, s);
    if (rc != V2A_OK) return rc;
    const long long SS = (long long)a.Dk * a.Dv;
    const uintptr_t at = (uintptr_t)p.dir[0].init | (uintptr_t)(p.ndir == 2 ? p.dir[1].init : nullptr);
    if (SS % 4 == 0 && (at & 15) == 0)
        hipLaunchKernelGGL((la_combine<4>), dim3(cdiv(SS, 256), (unsigned)(a.B * a.H), p.ndir), dim3(64), 0, s, p, pl.nseg, SS);
    else hipLaunchKernelGGL((la_combine<1>), dim3(cdiv(SS, 64), (unsigned)(a.B * a.H), p.ndir), dim3(64), 0, s, p, pl.nseg, SS);
    V2A_CHECK_LAUNCH();
    return V2A_OK;
}
// A recurrence over the whole sequence; the states before its segments are there
template <bool OUT> int la_recur(const LaArgs& a, LaScan p, const LaPlan& pl, int dtype, hipStream_t s) {
    p.ndir = 1;
    p.vst = a.Dv % 4 == 0 && (((uintptr_t)p.dir[0].init | (uintptr_t)p.last) & 15) == 0;      // the workspace is aligned
    p.NC = pl.NC; p.cps = pl.cps; p.nseg = pl.nseg; p.ndv = pl.ndv;
    return la_launch_scan<OUT>(a, p, pl.dvt, dtype, s);
}

struct LaFwdWs { size_t seg, decay, total; };
LaFwdWs la_fwd_ws(const LaPlan& p, size_t BH, size_t SS) {
    LaFwdWs w{};
    if (p.nseg > 1) {
        w.decay = la_up(BH * p.nseg * SS * 4);
        w.total = w.decay + la_up(BH * p.nseg * 4);
    }
    return w;
}
// Segments of two chunks: the states before the chunks come out of the local pass and the sum over segments, not of a further pass over k and v
bool la_pairs(const LaPlan& p) { return p.nseg > 1 && p.cps == 2; }
struct LaBwdWs { size_t seg, decay, seg2, decay2, sch, inner, inner_decay, q, k, v, part, total; };
LaBwdWs la_bwd_ws(const LaPlan& p, size_t B, size_t T, size_t H, int Hq, int Hk, int Hv, size_t Dk, size_t Dv, int per_token) {
    LaBwdWs w{};
    const size_t SS = Dk * Dv, BH = B * H, n = B * T * H;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at += la_up(bytes); return o; };
    w.seg = take(p.nseg > 1 ? BH * p.nseg * SS * 4 : 0);
    w.decay = take(p.nseg > 1 ? BH * p.nseg * 4 : 0);
    w.seg2 = take(p.nseg > 1 ? BH * p.nseg * SS * 4 : 0);
    w.decay2 = take(p.nseg > 1 ? BH * p.nseg * 4 : 0);
    w.sch = take(p.NC > 1 && !la_pairs(p) ? BH * p.NC * SS * 4 : 0);
    w.inner = take(la_pairs(p) ? BH * p.nseg * SS * 4 : 0);
    w.inner_decay = take(la_pairs(p) ? BH * p.nseg * 4 : 0);
    w.q = take((size_t)Hq < H ? n * Dk * 4 : 0);
    w.k = take((size_t)Hk < H ? n * Dk * 4 : 0);
    w.v = take((size_t)Hv < H ? n * Dv * 4 : 0);
    w.part = take(per_token ? 0 : BH * p.NC * 4);
    w.total = at;
    return w;
}

}  // namespace

extern "C" {

size_t v2a_linattn_fwd_workspace_bytes(int B, int T, int H, int Dk, int Dv, int dtype) {
    if (!la_dims(B, T, H, H, H, H, Dk, Dv, dtype) || B == 0) return 0;
    return la_fwd_ws(la_plan_fwd(B * H, T, Dk, Dv, dtype), (size_t)B * H, (size_t)Dk * Dv).total;
}

int v2a_linattn_fwd(const void* q, const void* k, const void* v, const float* g, const float* state, const int32_t* lens, void* out, float* state_out,
                    const int64_t* strides, int B, int T, int H, int Hq, int Hk, int Hv, int Dk, int Dv, int dtype, float scale, void* ws, size_t ws_bytes,
                    hipStream_t s) {
    if (!strides || !la_dims(B, T, H, Hq, Hk, Hv, Dk, Dv, dtype)) return V2A_ERR_ARG;
    if (B == 0 || (T == 0 && !state_out)) return V2A_OK;
    if (T > 0 && (!q || !k || !v || !g || !out)) return V2A_ERR_ARG;
    const LaPlan pl = la_plan_fwd(B * H, T, Dk, Dv, dtype);
    const LaFwdWs w = la_fwd_ws(pl, (size_t)B * H, (size_t)Dk * Dv);
    if (ws_bytes < w.total || (w.total && !ws)) return V2A_ERR_WORKSPACE;
    const LaArgs a = la_args(q, k, v, g, state, lens, nullptr, strides, B, T, H, Hq, Hk, Hv, Dk, Dv, scale);
    LaScan p{};
    LaDir& m = p.dir[0];
    m.init = state;
    m.seg = (float*)((char*)ws + w.seg);
    m.seg_decay = (float*)((char*)ws + w.decay);
    m.vx = la_vec(k, a.ks, B, T, Hk, Dk, dtype);
    m.vy = la_vec(v, a.vs, B, T, Hv, Dv, dtype);
    p.ndir = 1;
    p.last = state_out;
    p.out = out;
    p.vq = la_vec(q, a.qs, B, T, Hq, Dk, dtype);
    p.vo = Dv % (dtype == 0 ? 4 : 8) == 0 && ((uintptr_t)out & 15) == 0;
    if (pl.nseg > 1) {
        const int rc = la_segments(a, p, pl, dtype, s);
        if (rc != V2A_OK) return rc;
    }
    return la_recur<true>(a, p, pl, dtype, s);
}

size_t v2a_linattn_bwd_workspace_bytes(int B, int T, int H, int Hq, int Hk, int Hv, int Dk, int Dv, int dtype, int per_token_decay) {
    if (!la_dims(B, T, H, Hq, Hk, Hv, Dk, Dv, dtype)) return 0;
    return la_bwd_ws(la_plan_bwd(B * H, T, Dk, Dv, dtype), B, T, H, Hq, Hk, Hv, Dk, Dv, per_token_decay).total;
}

int v2a_linattn_bwd(const void* q, const void* k, const void* v, const float* g, const float* state, const int32_t* lens, const void* dout,
                    const float* dstate_out, void* dq, void* dk, void* dv, float* dg, float* dstate, const int64_t* strides, int B, int T, int H, int Hq, int Hk,
                    int Hv, int Dk, int Dv, int dtype, int per_token_decay, float scale, void* ws, size_t ws_bytes, hipStream_t s) {
    if (!strides || !la_dims(B, T, H, Hq, Hk, Hv, Dk, Dv, dtype)) return V2A_ERR_ARG;
    if (B > 0 && T > 0 && (!q || !k || !v || !g || !dout || !dq || !dk || !dv)) return V2A_ERR_ARG;
    const LaPlan pl = la_plan_bwd(B * H, T, Dk, Dv, dtype);
    const LaBwdWs w = la_bwd_ws(pl, B, T, H, Hq, Hk, Hv, Dk, Dv, per_token_decay);
    if (ws_bytes < w.total || (w.total && !ws)) return V2A_ERR_WORKSPACE;
    const LaArgs a = la_args(q, k, v, g, state, lens, dout, strides, B, T, H, Hq, Hk, Hv, Dk, Dv, scale);
    auto at = [&](size_t o) { return (float*)((char*)ws + o); };
    int rc = V2A_OK;
    if (B > 0) {
        const int vq = la_vec(q, a.qs, B, T, Hq, Dk, dtype), vk = la_vec(k, a.ks, B, T, Hk, Dk, dtype), vv = la_vec(v, a.vs, B, T, Hv, Dv, dtype);
        const int vd = la_vec(dout, a.ds, B, T, H, Dv, dtype);
        LaScan p{};
        p.dir[0] = LaDir{state, at(w.seg), at(w.decay), 0, vk, vv, 0};
        p.dir[1] = LaDir{dstate_out, at(w.seg2), at(w.decay2), 1, vq, vd, 0};
        if (pl.nseg > 1) {                   // states before the segments, and gradients of those behind them
            p.ndir = 2;
            if (la_pairs(pl)) { p.inner = at(w.inner); p.inner_decay = at(w.inner_decay); }
            rc = la_segments(a, p, pl, dtype, s);
            if (rc != V2A_OK) return rc;
        }
        if (pl.NC > 1 && !la_pairs(pl)) {    // states before the chunks
            p.chunk = at(w.sch);
            rc = la_recur<false>(a, p, pl, dtype, s);
            if (rc != V2A_OK) return rc;
        }
        if (T == 0 && dstate) {              // no tokens: the gradient passes through
            LaScan r{};
            r.dir[0] = p.dir[1]; r.last = dstate;
            rc = la_recur<false>(a, r, pl, dtype, s);
            if (rc != V2A_OK) return rc;
        }
        if (T > 0) {
            LaBwd d{};
            d.s_chunk[0] = at(la_pairs(pl) ? w.seg : w.sch); d.s_chunk[1] = at(la_pairs(pl) ? w.inner : w.sch);
            d.ns = la_pairs(pl) ? pl.nseg : pl.NC; d.shift = la_pairs(pl);
            d.s_first = state; d.e_last = dstate_out; d.e_seg = at(w.seg2); d.e_first = dstate;
            d.cps = pl.cps; d.nseg = pl.nseg;
            d.fq = Hq < H; d.fk = Hk < H; d.fv = Hv < H;
            d.dq = d.fq ? (void*)at(w.q) : dq;
            d.dk = d.fk ? (void*)at(w.k) : dk;
            d.dv = d.fv ? (void*)at(w.v) : dv;
            d.dg = per_token_decay ? dg : nullptr;
            d.dg_part = per_token_decay || !dg ? nullptr : at(w.part);
            d.NC = pl.NC; d.vq = vq; d.vk = vk; d.vv = vv; d.vd = vd;
            d.vst = Dv % 4 == 0 && (((uintptr_t)state | (uintptr_t)dstate_out | (uintptr_t)dstate) & 15) == 0;
            const dim3 grid((unsigned)((long long)B * H * pl.nseg));
            const int Dm = Dk > Dv ? Dk : Dv;
#define BWD(DT, D) hipLaunchKernelGGL((la_bwd_chunks<DT, D>), grid, dim3(4 * D * la_bwd_halves<DT, D>()), 0, s, a, d)
            if (Dm <= 32) { if (dtype == 0) BWD(0, 32); else if (dtype == 1) BWD(1, 32); else BWD(2, 32); }
            else if (Dm <= 64) { if (dtype == 0) BWD(3, 64); else if (dtype == 1) BWD(1, 64); else BWD(2, 64); }
            else if (Dm <= 96) { if (dtype == 0) BWD(0, 96); else if (dtype == 1) BWD(1, 96); else BWD(2, 96); }
            else { if (dtype == 0) BWD(0, 128); else if (dtype == 1) BWD(1, 128); else BWD(2, 128); }
#undef BWD
            V2A_CHECK_LAUNCH();
            const long long rows = (long long)B * T;
            const LaShares sh = {{{d.fq ? at(w.q) : nullptr, dq, Hq, H / Hq, Dk}, {d.fk ? at(w.k) : nullptr, dk, Hk, H / Hk, Dk},
                                  {d.fv ? at(w.v) : nullptr, dv, Hv, H / Hv, Dv}}};
#define CALL(DT) if (d.fq || d.fk || d.fv) hipLaunchKernelGGL((la_share<DT>), dim3(1024, 3), dim3(256), 0, s, sh, rows)
            LA_BY_TYPE(dtype, CALL);
#undef CALL
        }
    }
    if (dg && !per_token_decay) hipLaunchKernelGGL(la_dg_heads, dim3(H), dim3(256), 0, s, at(w.part), dg, (long long)B * pl.NC, H);
    V2A_CHECK_LAUNCH();
    return V2A_OK;
}

int v2a_linattn_step(const void* q, const void* k, const void* v, const float* g, float* state, const int32_t* slots, void* out, const int64_t* strides, int B,
                     int N, int H, int Hq, int Hk, int Hv, int Dk, int Dv, int dtype, float scale, hipStream_t s) {
    if (!strides || !la_dims(B, 1, H, Hq, Hk, Hv, Dk, Dv, dtype) || N < 0 || (!slots && N < B)) return V2A_ERR_ARG;
    if (B == 0) return V2A_OK;
    if (!q || !k || !v || !g || (!state && N > 0) || !out) return V2A_ERR_ARG;      // N = 0: every row is idle
    const int64_t* t = strides;
    const bool vec = Dv % 4 == 0 && ((uintptr_t)state & 15) == 0;
    int lv = 1;
    while (lv * (vec ? 4 : 1) < Dv) lv *= 2;
#define STEP(DT, W)                                                                                                                                     \
    hipLaunchKernelGGL((la_step_kernel<DT, W>), dim3(B * H), dim3(256), 0, s, q, k, v, g, state, slots, out, (long long)t[0], (long long)t[1],           \
                       (long long)t[2], (long long)t[3], (long long)t[4], (long long)t[5], (long long)t[6], (long long)t[7], B, N, H, Hq, Hk, Hv, Dk, Dv, lv, scale)
#define CALL(DT)              \
    if (vec) { STEP(DT, 4); } \
    else STEP(DT, 1)
    LA_BY_TYPE(dtype, CALL);
#undef CALL
#undef STEP
    V2A_CHECK_LAUNCH();
    return V2A_OK;
}

}  // extern "C"
