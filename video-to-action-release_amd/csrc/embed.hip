// Token embedding: out[i] = scale * table[id_i] + pos[i mod T], and its gradient: dtable[r] = scale * sum of dout over the tokens r,
// dpos[t] = sum over the sequences.  Ids outside [0, V) are empty: a zero row, no gradient.  Memory-bound: one read and one write per value.
//
// The gradient has no atomics and one order of summation: the tokens are sorted (stable: equal ids are neighbours, in token order), and fixed pieces of the sorted list are summed independently.
//   launch 1   sort (or the histogram of its first digit) in the first workgroups, dpos and the zero fill of dtable in the others, which need
//              no order and run beside it
//   (launches  further steps of the sort: two per digit where there are more than EM_SMALL tokens)
//   next       every piece of the list: rows that lie inside a piece are written, rows that cross a border leave fp32 partial sums
//   last       rows that cross borders: their partial sums, in piece order
#include "common.h"

namespace {

constexpr int EM_SORT_T = 1024, EM_WAVES = EM_SORT_T / 64, EM_KPT = 4, EM_SUB = EM_SORT_T * EM_KPT, EM_SMALL = 2 * EM_SUB, EM_BINS = 1024, EM_TILES = 32;

template <int DT> struct EmT { typedef unsigned short T; static constexpr int EPC = 8; };
template <> struct EmT<0> { typedef float T; static constexpr int EPC = 4; };
template <int DT> __device__ __forceinline__ float em_f(typename EmT<DT>::T x) {
    if constexpr (DT == 0) return x;
    else return v2a_h2f<DT == 2>(x);
}
template <int DT> __device__ __forceinline__ typename EmT<DT>::T em_r(float x) {
    if constexpr (DT == 0) return x;
    else return v2a_f2h<DT == 2>(x);
}
// W values from p[0 .. W): 16 bytes, or one value
template <int DT, int W> __device__ __forceinline__ void em_ld(const typename EmT<DT>::T* p, float* x) {
    if constexpr (W == 1) x[0] = em_f<DT>(*p);
    else if constexpr (DT == 0) {
        const float4 v = *(const float4*)p;
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else v2a_unpack_h8<DT == 2>(*(const uint4*)p, x);
}
template <int DT, int W> __device__ __forceinline__ void em_st(typename EmT<DT>::T* p, const float* x) {
    if constexpr (W == 1) *p = em_r<DT>(x[0]);
    else if constexpr (DT == 0) *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
    else *(uint4*)p = make_uint4(v2a_pack_h2<DT == 2>(x[0], x[1]), v2a_pack_h2<DT == 2>(x[2], x[3]), v2a_pack_h2<DT == 2>(x[4], x[5]), v2a_pack_h2<DT == 2>(x[6], x[7]));
}
// id of token i, or V for an empty place
__device__ __forceinline__ unsigned em_key(const void* ids, int wide, unsigned i, unsigned V) {
    if (wide) {
        const long long id = ((const long long*)ids)[i];
        return id >= 0 && id < (long long)V ? (unsigned)id : V;
    }
    const int id = ((const int*)ids)[i];
    return id >= 0 && (unsigned)id < V ? (unsigned)id : V;
}

struct EmShape {
    unsigned N, T, V;
    int D, lpr, ncol;      // lanes that share a row (power of two, at most 64), column blocks of lpr pieces
};

// A group of lpr lanes takes a row; each lane has RPT rows under way at once: 62891 rows of 384 fp32 from a table of 259 are written in 20 us
// (97 MB, 4.8 TB/s of writes), 8192 rows of 512 bf16 from 49408 in 7.5 us, 20 rows in 3.6 us (an empty launch: 3.7).
template <int DT, int W>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const void* ids, int wide, const void* table_, const void* pos_, void* out_, EmShape e, long long ldt,
                                                        long long ldp, float scale) {
    typedef typename EmT<DT>::T E;
    constexpr int RPT = 4;
    const E *table = (const E*)table_, *pos = (const E*)pos_;
    E* out = (E*)out_;
    const unsigned l = threadIdx.x & (e.lpr - 1), groups = gridDim.x * 256 / e.lpr, gid = (blockIdx.x * 256 + threadIdx.x) / e.lpr;
    for (unsigned long long r0 = gid; r0 < e.N; r0 += (unsigned long long)groups * RPT) {
        unsigned key[RPT];
#pragma unroll
        for (int j = 0; j < RPT; ++j) {
            const unsigned long long r = r0 + (unsigned long long)j * groups;
            key[j] = r < e.N ? em_key(ids, wide, (unsigned)r, e.V) : e.V;
        }
        for (int c = l * W; c < e.D; c += e.lpr * W) {
            float x[RPT][W];
#pragma unroll
            for (int j = 0; j < RPT; ++j)
                if (key[j] < e.V) em_ld<DT, W>(table + key[j] * ldt + c, x[j]);
#pragma unroll
            for (int j = 0; j < RPT; ++j) {
                const unsigned long long r = r0 + (unsigned long long)j * groups;
                if (r >= e.N) break;
                float p[W];
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    p[w] = 0.f;
                    x[j][w] = key[j] < e.V ? x[j][w] * scale : 0.f;
                }
                if (pos && key[j] < e.V) em_ld<DT, W>(pos + ((unsigned)r % e.T) * ldp + c, p);
                if (pos)
#pragma unroll
                    for (int w = 0; w < W; ++w) x[j][w] += p[w];
                em_st<DT, W>(out + r * e.D + c, x[j]);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------- sort
struct EmSort {
    const void* ids;
    int wide, bits, passes;                 // digits of `bits` bits, low first
    int split;                              // up to EM_SMALL tokens: low bits that name the workgroup
    unsigned N, V, tile, ntiles;            // tokens per workgroup of the many-workgroup form
    unsigned *key, *pos, *key2, *pos2;      // ping and pong
    unsigned* hist;                         // [ntiles][2^bits]
};

// Stable rank of each of this wave's 64 * kpt keys (key j of lane l is number 64 j + l) among the wave's equal digits, which also counts
// them: lanes with the digit's bits all equal find each other by ballots (a bit, drawn out over the word, against the ballot of it).
template <int KPT>
__device__ __forceinline__ void em_wave_rank(const unsigned (&dig)[KPT], const bool (&on)[KPT], int kpt, int bits, unsigned short* count, int lane, unsigned (&rank)[KPT]) {
#pragma unroll
    for (int j = 0; j < KPT; ++j) {
        if (j >= kpt) break;
        const unsigned long long all = __ballot(on[j]);
        unsigned lo = (unsigned)all, hi = (unsigned)(all >> 32);
        for (int b = 0; b < bits; ++b) {
            const int bit = (int)(dig[j] << (31 - b)) >> 31;
            const unsigned long long m = __ballot(bit);
            lo &= ~((unsigned)m ^ bit);
            hi &= ~((unsigned)(m >> 32) ^ bit);
        }
        const unsigned long long same = (unsigned long long)hi << 32 | lo;
        const unsigned below = __popcll(same & ((1ull << lane) - 1));
        const unsigned start = on[j] ? count[dig[j]] : 0u;
        rank[j] = start + below;
        __builtin_amdgcn_wave_barrier();
        if (on[j] && below == 0) count[dig[j]] = (unsigned short)(start + __popcll(same));
        __builtin_amdgcn_wave_barrier();
    }
}

// exclusive scan over the workgroup's 1024 threads
__device__ __forceinline__ unsigned em_scan(unsigned v, unsigned* tmp) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    unsigned x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    if (lane == 63) tmp[w] = x;
    __syncthreads();
    unsigned before = 0;
#pragma unroll
    for (int i = 0; i < EM_WAVES; ++i) {      // all read at once
        const unsigned t = tmp[i];
        before += i < w ? t : 0u;
    }
    __syncthreads();
    return before + x - v;
}

// this thread's digit: counts of the waves -> counts of the waves before each; returns their sum
__device__ __forceinline__ unsigned em_waves_scan(unsigned short (*count)[EM_BINS]) {
    unsigned c[EM_WAVES], n = 0;
#pragma unroll
    for (int i = 0; i < EM_WAVES; ++i) c[i] = count[i][threadIdx.x];
#pragma unroll
    for (int i = 0; i < EM_WAVES; ++i) {
        count[i][threadIdx.x] = (unsigned short)n;
        n += c[i];
    }
    return n;
}

struct EmSortLds {
    unsigned short count[EM_WAVES][EM_BINS];
    unsigned base[EM_BINS], tmp[EM_WAVES];
};

// Up to EM_SMALL tokens: a workgroup takes those whose id ends in the bits `blk`, lays them behind the tokens of the workgroups before it
// (equal ids have to meet, not to be in order) and sorts them by the other bits, all digits through LDS.  Empty places go with the last workgroup,
// whose largest ids they are.  Bound by the six vector instructions per key and bit of the ballots: 8192 tokens of 49408 rows, half of them one,
// take 11.5 us (17.3 by one workgroup with two digits); with a zero fill of 51 MB beside it 15.
__device__ void em_sort_small(const EmSort& s, EmSortLds& L, unsigned (*xch)[EM_SMALL], unsigned blk) {
    constexpr int KPT = EM_SMALL / EM_SORT_T;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, bins = 1 << s.bits;
    const unsigned last = (1u << s.split) - 1;
    unsigned key[KPT], pos[KPT], n = s.N, start = 0;
    bool on[KPT];
    int kpt = (n + EM_SORT_T - 1) / EM_SORT_T;
    auto place = [&](int j) { return (unsigned)(w * 64 * kpt + j * 64 + lane); };
#pragma unroll
    for (int j = 0; j < KPT; ++j) {
        const unsigned i = place(j);
        on[j] = j < kpt && i < n;
        pos[j] = i;
        key[j] = on[j] ? em_key(s.ids, s.wide, i, s.V) : 0u;
    }
    if (s.split) {
        unsigned own = 0, low = 0;
        unsigned long long mine[KPT];
#pragma unroll
        for (int j = 0; j < KPT; ++j) {
            const unsigned b = key[j] == s.V ? last : key[j] & last;
            mine[j] = __ballot(on[j] && b == blk);
            own += __popcll(mine[j]);
            low += __popcll(__ballot(on[j] && b < blk));
        }
        if (lane == 0) L.tmp[w] = own | low << 16;
        __syncthreads();
        unsigned at = 0, sum = 0;
#pragma unroll
        for (int i = 0; i < EM_WAVES; ++i) {
            const unsigned t = L.tmp[i];
            at += i < w ? t & 0xffffu : 0u;
            sum += t;
        }
        n = sum & 0xffffu;
        start = sum >> 16;
        if (n == 0) return;
#pragma unroll
        for (int j = 0; j < KPT; ++j) {
            if (mine[j] >> lane & 1) {
                const unsigned d = at + __popcll(mine[j] & ((1ull << lane) - 1));
                xch[0][d] = key[j];
                xch[1][d] = pos[j];
            }
            at += __popcll(mine[j]);
        }
        kpt = (n + EM_SORT_T - 1) / EM_SORT_T;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < KPT; ++j) {
            const unsigned i = place(j);
            on[j] = j < kpt && i < n;
            key[j] = on[j] ? xch[0][i] : 0u;
            pos[j] = on[j] ? xch[1][i] : 0u;
        }
    }
    for (int p = 0; p < s.passes; ++p) {
        for (int i = threadIdx.x; i < EM_WAVES * EM_BINS / 2; i += EM_SORT_T) ((unsigned*)L.count)[i] = 0u;
        __syncthreads();
        unsigned dig[KPT], rank[KPT];
#pragma unroll
        for (int j = 0; j < KPT; ++j) dig[j] = (key[j] >> (s.split + p * s.bits)) & (bins - 1);
        em_wave_rank(dig, on, kpt, s.bits, L.count[w], lane, rank);
        __syncthreads();
        unsigned total = 0;
        if (threadIdx.x < bins)
            total = em_waves_scan(L.count);
        L.base[threadIdx.x] = em_scan(total, L.tmp);
        __syncthreads();
        const bool done = p == s.passes - 1;      // the last places are the list's
#pragma unroll
        for (int j = 0; j < KPT; ++j)
            if (on[j]) {
                const unsigned d = L.base[dig[j]] + L.count[w][dig[j]] + rank[j];
                if (done) {
                    s.key[start + d] = key[j];
                    s.pos[start + d] = pos[j];
                } else {
                    xch[0][d] = key[j];
                    xch[1][d] = pos[j];
                }
            }
        if (done) return;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < KPT; ++j)
            if (on[j]) {
                const unsigned i = place(j);
                key[j] = xch[0][i];
                pos[j] = xch[1][i];
            }
        __syncthreads();
    }
}

// How many tokens of workgroup `t`'s tile have each digit of pass p.  (Counted by the scatter of the digit before, with atomics on the tile
// that a token goes to, it would save a launch of 5 us, but a token that fills half the list takes 50 us at one address.)
__device__ void em_hist(const EmSort& s, int p, unsigned t, unsigned* count) {
    const int bins = 1 << s.bits;
    for (int i = threadIdx.x; i < bins; i += EM_SORT_T) count[i] = 0u;
    __syncthreads();
    const unsigned a = t * s.tile, b = s.N - a < s.tile ? s.N : a + s.tile;
    for (unsigned i = a + threadIdx.x; i < b; i += EM_SORT_T) {
        const unsigned k = p == 0 ? em_key(s.ids, s.wide, i, s.V) : s.key[i];
        atomicAdd(&count[(k >> (p * s.bits)) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < bins; i += EM_SORT_T) s.hist[(size_t)t * bins + i] = count[i];
}
__global__ __launch_bounds__(EM_SORT_T) void embed_hist_kernel(EmSort s, int p) {
    __shared__ unsigned count[EM_BINS];
    em_hist(s, p, blockIdx.x, count);
}
// the tokens of a tile to their places of pass p; a workgroup adds up the at most EM_TILES histograms itself.  62891 tokens, 9 bits:
// 8.4 us in tiles of 2048, 9.1 in 1024, 10.4 in 4096
__global__ __launch_bounds__(EM_SORT_T) void embed_scatter_kernel(EmSort s, int p) {
    __shared__ EmSortLds L;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, bins = 1 << s.bits;
    unsigned before = 0, total = 0;
    if (threadIdx.x < bins)
        for (unsigned t0 = 0; t0 < s.ntiles; t0 += 16) {
            unsigned n[16];
#pragma unroll
            for (unsigned j = 0; j < 16; ++j) n[j] = t0 + j < s.ntiles ? s.hist[(size_t)(t0 + j) * bins + threadIdx.x] : 0u;
#pragma unroll
            for (unsigned j = 0; j < 16; ++j) {
                if (t0 + j < blockIdx.x) before += n[j];
                total += n[j];
            }
        }
    const unsigned start = em_scan(total, L.tmp) + before;
    L.base[threadIdx.x] = start;
    const unsigned a = blockIdx.x * s.tile, end = s.N - a < s.tile ? s.N : a + s.tile;
    const int kpt = s.tile < (unsigned)EM_SUB ? s.tile / EM_SORT_T : EM_KPT;
    for (unsigned a0 = a; a0 < end; a0 += EM_SUB) {
        for (int i = threadIdx.x; i < EM_WAVES * EM_BINS / 2; i += EM_SORT_T) ((unsigned*)L.count)[i] = 0u;
        unsigned key[EM_KPT], pos[EM_KPT], dig[EM_KPT], rank[EM_KPT];
        bool on[EM_KPT];
#pragma unroll
        for (int j = 0; j < EM_KPT; ++j) {
            const unsigned i = a0 + w * 64 * kpt + j * 64 + lane;
            on[j] = j < kpt && i < end;
            key[j] = !on[j] ? 0u : p == 0 ? em_key(s.ids, s.wide, i, s.V) : s.key[i];
            pos[j] = !on[j] ? 0u : p == 0 ? i : s.pos[i];
            dig[j] = (key[j] >> (p * s.bits)) & (bins - 1);
        }
        __syncthreads();
        em_wave_rank(dig, on, kpt, s.bits, L.count[w], lane, rank);
        __syncthreads();
        unsigned n = 0;
        if (threadIdx.x < bins)
            n = em_waves_scan(L.count);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < EM_KPT; ++j)
            if (on[j]) {
                const unsigned d = L.base[dig[j]] + L.count[w][dig[j]] + rank[j];
                s.key2[d] = key[j];
                s.pos2[d] = pos[j];
            }
        __syncthreads();
        if (threadIdx.x < bins) L.base[threadIdx.x] += n;
    }
}

// ---------------------------------------------------------------------------------------------------------------------- gradient
struct EmGrad {
    const void* dout;
    void *dtable, *dpos;
    unsigned P, nsort, nfill;      // rows of dpos; workgroups of launch 1 that sort / fill (those between the two compute dpos)
    float scale;
};

// Launch 1.  dpos: one workgroup per (position, column block); wave w adds sequences w, w + 16, .., the waves' sums are added in order.
template <int DT, int W>
__global__ __launch_bounds__(EM_SORT_T) void embed_first_kernel(EmSort s, EmGrad g, EmShape e) {
    typedef typename EmT<DT>::T E;
    __shared__ union {
        struct { EmSortLds l; unsigned xch[2][EM_SMALL]; } sort;
        unsigned count[EM_BINS];
        float part[EM_WAVES][64 * W];
    } sm;
    if (blockIdx.x < g.nsort) {
        if (s.N <= (unsigned)EM_SMALL) em_sort_small(s, sm.sort.l, sm.sort.xch, blockIdx.x);
        else em_hist(s, 0, blockIdx.x, sm.count);
        return;
    }
    const unsigned blk = blockIdx.x - g.nsort, ndpos = gridDim.x - g.nsort - g.nfill;
    if (blk >= ndpos) {
        const size_t n = (size_t)e.V * e.D;
        E* q = (E*)g.dtable;
        const size_t step = (size_t)g.nfill * EM_SORT_T, at = (size_t)(blk - ndpos) * EM_SORT_T + threadIdx.x;
        if (((uintptr_t)q & 15) == 0) {
            const size_t nv = n / EmT<DT>::EPC;
            for (size_t i = at; i < nv; i += step) ((uint4*)q)[i] = make_uint4(0u, 0u, 0u, 0u);
            for (size_t i = nv * EmT<DT>::EPC + at; i < n; i += step) q[i] = 0;
        } else
            for (size_t i = at; i < n; i += step) q[i] = 0;
        return;
    }
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const unsigned nc = (e.D + 64 * W - 1) / (64 * W), Bn = e.N / e.T;
    for (unsigned long long u = blk; u < (unsigned long long)g.P * nc; u += ndpos) {
        const unsigned t = (unsigned)(u / nc);
        const int c = (int)(u % nc) * 64 * W + lane * W;
        float acc[W];
#pragma unroll
        for (int i = 0; i < W; ++i) acc[i] = 0.f;
        if (t < e.T && c < e.D)
            for (unsigned b0 = w; b0 < Bn; b0 += 4 * EM_WAVES) {
                float x[4][W];
                bool on[4];
#pragma unroll
                for (unsigned j = 0; j < 4; ++j) {
                    const unsigned b = b0 + j * EM_WAVES;
                    on[j] = b < Bn && em_key(s.ids, s.wide, b * e.T + t, e.V) < e.V;
                }
#pragma unroll
                for (unsigned j = 0; j < 4; ++j)
                    if (on[j]) em_ld<DT, W>((const E*)g.dout + (size_t)((b0 + j * EM_WAVES) * e.T + t) * e.D + c, x[j]);
#pragma unroll
                for (unsigned j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < W; ++i) acc[i] += on[j] ? x[j][i] : 0.f;
            }
#pragma unroll
        for (int i = 0; i < W; ++i) sm.part[w][i * 64 + lane] = acc[i];
        __syncthreads();
        if (w == 0 && c < e.D) {
            for (int j = 1; j < EM_WAVES; ++j)
#pragma unroll
                for (int i = 0; i < W; ++i) acc[i] += sm.part[j][i * 64 + lane];
            em_st<DT, W>((E*)g.dpos + (size_t)t * e.D + c, acc);
        }
        __syncthreads();
    }
}

// Pieces of `ts` neighbours of the sorted list, one per group of lpr lanes.  part [pieces][2][Dp]: 0 = a row that began before the piece
// (through to its end or past the piece), 1 = a row that begins inside and goes on behind it.  Bound by the read of dout: 62891 rows of 384 fp32
// in 21.6 us (4.5 TB/s), 8192 rows of 512 bf16 in 7.7.
template <int DT, int W>
__global__ __launch_bounds__(256) void embed_pieces_kernel(const unsigned* key, const unsigned* pos, EmGrad g, EmShape e, float* part, int Dp, unsigned ts) {
    typedef typename EmT<DT>::T E;
    constexpr int AHEAD = 8;
    const unsigned l = threadIdx.x & (e.lpr - 1);
    const unsigned long long gid = ((unsigned long long)blockIdx.x * 256 + threadIdx.x) / e.lpr;
    const unsigned long long t = gid / e.ncol, a64 = t * ts;
    if (a64 >= e.N) return;
    const int c = ((int)(gid % e.ncol) * e.lpr + l) * W;
    if (c >= e.D) return;
    const unsigned a = (unsigned)a64, b = e.N - a < ts ? e.N : a + ts;
    unsigned cur = key[a];
    bool before = a > 0 && key[a - 1] == cur;
    float acc[W];
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] = 0.f;
    auto partial = [&](int which) {
        float* q = part + (t * 2 + which) * Dp + c;
        if constexpr (W == 1) q[0] = acc[0];
        else
#pragma unroll
            for (int i = 0; i < W; i += 4) *(float4*)(q + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
    };
    auto whole = [&]() {
        float x[W];
#pragma unroll
        for (int i = 0; i < W; ++i) x[i] = acc[i] * g.scale;
        em_st<DT, W>((E*)g.dtable + (size_t)cur * e.D + c, x);
    };
    unsigned k[AHEAD], r[AHEAD];
    auto fetch = [&](unsigned i0) {          // pieces begin at multiples of eight, and the lists have room to the next one
        const uint4 k0 = *(const uint4*)(key + i0), k1 = *(const uint4*)(key + i0 + 4), r0 = *(const uint4*)(pos + i0), r1 = *(const uint4*)(pos + i0 + 4);
        k[0] = k0.x; k[1] = k0.y; k[2] = k0.z; k[3] = k0.w; k[4] = k1.x; k[5] = k1.y; k[6] = k1.z; k[7] = k1.w;
        r[0] = r0.x; r[1] = r0.y; r[2] = r0.z; r[3] = r0.w; r[4] = r1.x; r[5] = r1.y; r[6] = r1.z; r[7] = r1.w;
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (i0 + j >= b) k[j] = e.V;
    };
    fetch(a);
    for (unsigned i0 = a; i0 < b && cur < e.V; i0 += AHEAD) {
        float x[AHEAD][W];
        unsigned kk[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            kk[j] = k[j];
            if (kk[j] < e.V) em_ld<DT, W>((const E*)g.dout + (size_t)r[j] * e.D + c, x[j]);
        }
        if (i0 + AHEAD < b) fetch(i0 + AHEAD);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (i0 + j >= b) break;
            if (kk[j] != cur) {
                if (before) partial(0);
                else if (cur < e.V) whole();
                before = false;
                cur = kk[j];
#pragma unroll
                for (int i = 0; i < W; ++i) acc[i] = 0.f;
            }
            if (kk[j] < e.V)
#pragma unroll
                for (int i = 0; i < W; ++i) acc[i] += x[j][i];
        }
    }
    if (cur >= e.V) return;
    if (before) partial(0);
    else if (b < e.N && key[b] == cur) partial(1);
    else whole();
}

// Rows that cross pieces: the piece in which one begins adds its part 1 and the parts 0 of the pieces behind it, in order.  One wave per
// (piece, 256 columns), most of which have nothing to do; a run's end is found first, 64 borders at a time, so that the sum has known bounds and
// loads under way.  Runs over more than EM_LONG pieces are left to the whole workgroup: wave w adds pieces w, w + 16, .., the sums of the waves
// in order.  (All runs by the workgroup, one after the other, took 22 us where many short ones lie close together, against 8 to 9, most
// of it the launch and the dependent reads before the sum.)
constexpr int EM_JOIN = 16, EM_LONG = 32;
template <int DT>
__global__ __launch_bounds__(64 * EM_JOIN) void embed_join_kernel(const unsigned* key, EmGrad g, EmShape e, const float* part, int Dp, unsigned ts) {
    typedef typename EmT<DT>::T E;
    __shared__ float sum[EM_JOIN][256];
    __shared__ unsigned ends[EM_JOIN], ids[EM_JOIN];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned np = (e.N - 1) / ts + 1;
    const unsigned long long t = (unsigned long long)blockIdx.x * EM_JOIN + w, a = t * ts, b = a + ts;
    const int c0 = blockIdx.y * 256, c = c0 + lane * 4;
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [](float4& s, const float4& x) { s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w; };
    // parts 0 of pieces i, i + step, .. before `to`, eight under way; places behind `to` load the last piece again and leave it out
    auto sums = [&](float4& s, unsigned i, unsigned to, unsigned step) {
        for (; i < to; i += 8 * step) {
            float4 x[8];
#pragma unroll
            for (unsigned j = 0; j < 8; ++j) {
                const unsigned k = i + j * step;
                x[j] = *(const float4*)(part + (size_t)(k < to ? k : to - 1) * 2 * Dp + c);
            }
#pragma unroll
            for (unsigned j = 0; j < 8; ++j) add(s, i + j * step < to ? x[j] : zero);
        }
    };
    unsigned end = 0, cur = 0;
    if (b < e.N) {
        cur = key[b - 1];
        const bool owns = cur < e.V && key[b] == cur && !(key[a] == cur && a > 0 && key[a - 1] == cur);
        if (owns) {
            unsigned lo = (unsigned)t + 2, hi = np;      // the first piece from t + 2 on that begins with another id lies in [lo, hi]
            while (lo < hi) {
                const unsigned step = (hi - lo + 63) / 64, i = lo + lane * step;
                const unsigned n = __popcll(__ballot(i < hi && key[(size_t)i * ts] == cur));      // sorted: a prefix of the probes
                if (n == 0) { hi = lo; break; }
                const unsigned top = lo + n * step;
                lo = lo + (n - 1) * step + 1;
                hi = top < hi ? top : hi;
            }
            end = hi;
        }
    }
    const bool wide = end > t + 1 + EM_LONG;
    if (lane == 0) { ends[w] = wide ? end : 0u; ids[w] = cur; }
    if (end && !wide && c < e.D) {
        float4 s = *(const float4*)(part + (t * 2 + 1) * Dp + c);
        sums(s, (unsigned)t + 1, __builtin_amdgcn_readfirstlane(end), 1);
        const float x[4] = {s.x, s.y, s.z, s.w};
        E* q = (E*)g.dtable + (size_t)cur * e.D + c;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (c + r < e.D) q[r] = em_r<DT>(x[r] * g.scale);
    }
    __syncthreads();
    for (unsigned long long left = __ballot(lane < EM_JOIN && ends[lane & (EM_JOIN - 1)] != 0); left; left &= left - 1) {
        const int o = __ffsll(left) - 1;
        const size_t t0 = (size_t)blockIdx.x * EM_JOIN + o;
        float4 s = zero;
        if (c < e.D) {
            if (w == 0) s = *(const float4*)(part + (t0 * 2 + 1) * Dp + c);
            sums(s, (unsigned)t0 + 1 + w, __builtin_amdgcn_readfirstlane(ends[o]), EM_JOIN);
        }
        *(float4*)&sum[w][lane * 4] = s;
        __syncthreads();
        const int d = threadIdx.x;
        if (d < 256 && c0 + d < e.D) {
            float y = sum[0][d];
#pragma unroll
            for (int i = 1; i < EM_JOIN; ++i) y += sum[i][d];
            ((E*)g.dtable)[(size_t)ids[o] * e.D + c0 + d] = em_r<DT>(y * g.scale);
        }
        __syncthreads();
    }
}

bool em_dims(long long N, long long T, long long V, int D, int dtype) {
    return N >= 0 && N < (1ll << 31) && T > 0 && N % T == 0 && V > 0 && V < (1ll << 31) - 1 && D > 0 && dtype >= 0 && dtype <= 2;
}
EmShape em_shape(long long N, long long T, long long V, int D, int W) {
    EmShape e;
    e.N = (unsigned)N; e.T = (unsigned)(T < (1ll << 31) ? T : (1ll << 31)); e.V = (unsigned)V; e.D = D;
    const int pieces = cdiv(D, W);
    e.lpr = 1;
    while (e.lpr < pieces && e.lpr < 64) e.lpr *= 2;
    // 64 lanes would idle in the last block of a row of, say, 96 pieces: half of them where that covers fewer places
    while (e.lpr > 16 && cdiv(pieces, e.lpr / 2) * (e.lpr / 2) < cdiv(pieces, e.lpr) * e.lpr) e.lpr /= 2;
    e.ncol = cdiv(pieces, e.lpr);
    return e;
}
// pieces of 8 .. 64 tokens: long ones leave fewer partial sums, but a few thousand lane groups are needed to keep the memory busy
unsigned em_piece(long long N, int D, int dtype) {
    const long long ncol = cdiv(D, dtype == 0 ? 256 : 512);
    unsigned ts = 8;
    while (ts < 64 && N * ncol / (ts * 2) >= 4096) ts *= 2;
    return ts;
}
// Bits by which up to EM_SMALL tokens are shared out among workgroups: so many that one digit is left, and three where a workgroup alone would
// have several tokens a thread (8192 tokens, 300 ids: 11.5 us against 12.7)
int em_split(long long N, int bits) {
    const int one = bits <= 10 ? 0 : bits < 16 ? bits - 10 : 6, share = N > EM_SORT_T && bits > 3 ? 3 : 0;
    return one > share ? one : share;
}
struct EmWs { size_t key, pos, key2, pos2, hist, part, total; int Dp; unsigned ts; };
EmWs em_ws(long long N, int D, int dtype) {
    EmWs w;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t o = at; at += (n + 255) & ~(size_t)255; return o; };
    w.ts = em_piece(N, D, dtype);
    w.Dp = (D + 7) & ~7;
    const size_t n4 = (size_t)(N + 7) / 8 * 8 * 4;
    w.key = take(n4); w.pos = take(n4);
    w.key2 = take(N > EM_SMALL ? n4 : 0); w.pos2 = take(N > EM_SMALL ? n4 : 0);
    w.hist = take(N > EM_SMALL ? (size_t)EM_TILES * EM_BINS * 4 : 0);
    w.part = take((size_t)cdiv(N, w.ts) * 2 * w.Dp * 4);
    w.total = at;
    return w;
}
bool em_al(const void* p, long long ld, int dtype) { return ((uintptr_t)p & 15) == 0 && ld * (dtype == 0 ? 4 : 2) % 16 == 0; }

#define EM_BY_TYPE(dtype, vec, CALL)                          \
    do {                                                      \
        if ((dtype) == 0) { if (vec) { CALL(0, 4); } else { CALL(0, 1); } } \
        else if ((dtype) == 1) { if (vec) { CALL(1, 8); } else { CALL(1, 1); } } \
        else { if (vec) { CALL(2, 8); } else { CALL(2, 1); } } \
    } while (0)

}  // namespace

extern "C" {

int v2a_embed_fwd(const void* ids, int ids64, const void* table, const void* pos, void* out, long long N, long long T, long long V, int D, long long ld_table,
                  long long ld_pos, int dtype, float scale, hipStream_t s) {
    if (!em_dims(N, T, V, D, dtype) || ld_table < 0 || ld_pos < 0) return V2A_ERR_ARG;
    if (N == 0) return V2A_OK;
    if (!ids || !table || !out) return V2A_ERR_ARG;
    const bool vec = em_al(table, V > 1 ? ld_table : 0, dtype) && em_al(out, D, dtype) && (!pos || em_al(pos, T > 1 ? ld_pos : 0, dtype));
    const EmShape e = em_shape(N, T, V, D, vec ? (dtype == 0 ? 4 : 8) : 1);
    long long blocks = (N * e.lpr + 1023) / 1024;
    if (blocks > 8192) blocks = 8192;
    if (blocks < 256) blocks = (N * e.lpr + 255) / 256;      // few rows: one each
#define CALL(DT, W) hipLaunchKernelGGL((embed_fwd_kernel<DT, W>), dim3((unsigned)blocks), dim3(256), 0, s, ids, ids64, table, pos, out, e, ld_table, ld_pos, scale)
    EM_BY_TYPE(dtype, vec, CALL);
#undef CALL
    V2A_CHECK_LAUNCH();
    return V2A_OK;
}

size_t v2a_embed_bwd_workspace_bytes(long long N, long long V, int D, int dtype) {
    if (!em_dims(N, 1, V, D, dtype) || N == 0) return 0;
    return em_ws(N, D, dtype).total;
}

int v2a_embed_bwd(const void* ids, int ids64, const void* dout, void* dtable, void* dpos, long long N, long long T, long long V, int D, long long pos_rows, int dtype,
                  float scale, void* ws, size_t ws_bytes, hipStream_t s) {
    if (!em_dims(N, T, V, D, dtype) || !dtable || (dpos && (pos_rows < T || pos_rows >= (1ll << 31)) && N > 0)) return V2A_ERR_ARG;
    if (N > 0 && (!ids || !dout)) return V2A_ERR_ARG;
    const EmWs w = em_ws(N, D, dtype);
    if (N > 0 && (ws_bytes < w.total || !ws)) return V2A_ERR_WORKSPACE;
    char* base = (char*)ws;
    const bool vec = em_al(dout, D, dtype) && em_al(dtable, D, dtype) && em_al(dpos, D, dtype);
    const EmShape e = em_shape(N, T, V, D, vec ? (dtype == 0 ? 4 : 8) : 1);
    EmSort q{};
    q.ids = ids; q.wide = ids64; q.N = (unsigned)N; q.V = (unsigned)V;
    int bits = 1;
    while ((V >> bits) > 0) ++bits;               // keys 0 .. V
    if (N <= EM_SMALL) q.split = em_split(N, bits);
    bits -= q.split;
    q.passes = cdiv(bits, 10);
    q.bits = cdiv(bits, q.passes);
    q.key = (unsigned*)(base + w.key); q.pos = (unsigned*)(base + w.pos);
    q.key2 = (unsigned*)(base + w.key2); q.pos2 = (unsigned*)(base + w.pos2);
    q.hist = (unsigned*)(base + w.hist);
    q.tile = EM_SORT_T;
    while (cdiv(N, q.tile) > EM_TILES) q.tile *= 2;
    q.ntiles = cdiv(N, q.tile);
    EmGrad g{};
    g.dout = dout; g.dtable = dtable; g.dpos = dpos; g.scale = scale;
    g.P = dpos ? (unsigned)pos_rows : 0u;
    g.nsort = N == 0 ? 0 : N <= EM_SMALL ? 1 << q.split : q.ntiles;
    const int W = vec ? (dtype == 0 ? 4 : 8) : 1;
    const long long units = (long long)g.P * cdiv(D, 64 * W), ndpos = units < 4096 ? units : 4096;
    const long long fill = ((long long)V * D * (dtype == 0 ? 4 : 2) + 65535) / 65536;
    g.nfill = (unsigned)(fill < 1024 ? fill : 1024);
#define CALL(DT, W) hipLaunchKernelGGL((embed_first_kernel<DT, W>), dim3(g.nsort + (unsigned)ndpos + g.nfill), dim3(EM_SORT_T), 0, s, q, g, e)
    EM_BY_TYPE(dtype, vec, CALL);
#undef CALL
    V2A_CHECK_LAUNCH();
    if (N == 0) return V2A_OK;
    if (N > EM_SMALL) {
        for (int p = 0; p < q.passes; ++p) {
            if (p > 0) hipLaunchKernelGGL(embed_hist_kernel, dim3(q.ntiles), dim3(EM_SORT_T), 0, s, q, p);
            hipLaunchKernelGGL(embed_scatter_kernel, dim3(q.ntiles), dim3(EM_SORT_T), 0, s, q, p);
            unsigned* t = q.key; q.key = q.key2; q.key2 = t;
            t = q.pos; q.pos = q.pos2; q.pos2 = t;
        }
        V2A_CHECK_LAUNCH();
    }
    const unsigned pieces = (unsigned)cdiv(N, w.ts);
    const long long lanes = (long long)pieces * e.ncol * e.lpr;
#define CALL(DT, W) hipLaunchKernelGGL((embed_pieces_kernel<DT, W>), dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, s, q.key, q.pos, g, e, (float*)(base + w.part), w.Dp, w.ts)
    EM_BY_TYPE(dtype, vec, CALL);
#undef CALL
    V2A_CHECK_LAUNCH();
    if (pieces > 1) {
#define CALL(DT, W) hipLaunchKernelGGL((embed_join_kernel<DT>), dim3(cdiv(pieces - 1, EM_JOIN), cdiv(D, 256)), dim3(64 * EM_JOIN), 0, s, q.key, g, e, (const float*)(base + w.part), w.Dp, w.ts)
        EM_BY_TYPE(dtype, false, CALL);
#undef CALL
        V2A_CHECK_LAUNCH();
    }
    return V2A_OK;
}

}  // extern "C"
