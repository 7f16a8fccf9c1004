// Token embedding: out[i] = scale * table[id_i] + pos[i mod T], and its gradient: dtable[r] = scale * sum of dout over the tokens r in order,
// dpos[t] = sum over the sequences.  Ids outside [0, V) are empty: a zero row, no gradient.
#include "common.h"

namespace {

template <int DT> __device__ __forceinline__ float em_ld(const void* p, long long i) {
    if constexpr (DT == 0) return ((const float*)p)[i];
    else return v2a_h2f<DT == 2>(((const unsigned short*)p)[i]);
}
template <int DT> __device__ __forceinline__ void em_st(void* p, long long i, float x) {
    if constexpr (DT == 0) ((float*)p)[i] = x;
    else ((unsigned short*)p)[i] = v2a_f2h<DT == 2>(x);
}
__device__ __forceinline__ long long em_id(const void* ids, int wide, long long i) { return wide ? ((const long long*)ids)[i] : (long long)((const int*)ids)[i]; }

template <int DT>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const void* ids, int wide, const void* table, const void* pos, void* out, long long N, long long T, long long V, int D,
                                                        long long ldt, long long ldp, float scale) {
    for (long long i = blockIdx.x; i < N; i += gridDim.x) {
        const long long id = em_id(ids, wide, i);
        for (int c = threadIdx.x; c < D; c += 256) {
            float y = 0.f;
            if (id >= 0 && id < V) {
                y = em_ld<DT>(table, id * ldt + c) * scale;
                if (pos) y += em_ld<DT>(pos, (i % T) * ldp + c);
            }
            em_st<DT>(out, i * D + c, y);
        }
    }
}

template <int DT>
__global__ __launch_bounds__(256) void embed_bwd_simple(const void* ids, int wide, const void* dout, void* dtable, long long N, long long V, int D,
                                                        float scale) {
    __shared__ int hit[256];
    for (long long r = blockIdx.x; r < V; r += gridDim.x)
    for (int c0 = 0; c0 < D; c0 += 256) {
        const int c = c0 + threadIdx.x;
        float s = 0.f;
        for (long long i0 = 0; i0 < N; i0 += 256) {
            const long long i = i0 + threadIdx.x;
            const int m = i < N && em_id(ids, wide, i) == r;
            if (!__syncthreads_or(m)) continue;
            hit[threadIdx.x] = m;
            __syncthreads();
            for (int j = 0; j < 256; ++j)
                if (hit[j] && c < D) s += em_ld<DT>(dout, (i0 + j) * D + c);
            __syncthreads();
        }
        if (c < D) em_st<DT>(dtable, r * D + c, s * scale);
    }
}

template <int DT>
__global__ __launch_bounds__(256) void embed_dpos_kernel(const void* ids, int wide, const void* dout, void* dpos, long long Bn, long long T, long long V, int D, long long P) {
    for (long long t = blockIdx.x; t < P; t += gridDim.x)
    for (int c = threadIdx.x; c < D; c += 256) {
        float s = 0.f;
        if (t < T)
            for (long long b = 0; b < Bn; ++b) {
                const long long id = em_id(ids, wide, b * T + t);
                if (id >= 0 && id < V) s += em_ld<DT>(dout, (b * T + t) * D + c);
            }
        em_st<DT>(dpos, t * D + c, s);
    }
}

#define EM_BY_TYPE(dtype, CALL)        \
    do {                               \
        if ((dtype) == 0) { CALL(0); } \
        else if ((dtype) == 1) { CALL(1); } \
        else { CALL(2); }              \
    } while (0)

bool em_dims(long long N, long long T, long long V, int D, int dtype) {
    return N >= 0 && N < (1ll << 31) && T > 0 && N % T == 0 && V > 0 && V < (1ll << 31) - 1 && D > 0 && dtype >= 0 && dtype <= 2;
}

}  // namespace

extern "C" {

int v2a_embed_fwd(const void* ids, int ids64, const void* table, const void* pos, void* out, long long N, long long T, long long V, int D, long long ld_table,
                  long long ld_pos, int dtype, float scale, hipStream_t s) {
    if (!em_dims(N, T, V, D, dtype) || ld_table < 0 || ld_pos < 0) return V2A_ERR_ARG;
    if (N == 0) return V2A_OK;
    if (!ids || !table || !out) return V2A_ERR_ARG;
#define CALL(DT) hipLaunchKernelGGL((embed_fwd_kernel<DT>), dim3((unsigned)(N < 65536 ? N : 65536)), dim3(256), 0, s, ids, ids64, table, pos, out, N, T, V, D, ld_table, ld_pos, scale)
    EM_BY_TYPE(dtype, CALL);
#undef CALL
    V2A_CHECK_LAUNCH();
    return V2A_OK;
}

size_t v2a_embed_bwd_workspace_bytes(long long N, long long V, int D) { return 0; }

int v2a_embed_bwd(const void* ids, int ids64, const void* dout, void* dtable, void* dpos, long long N, long long T, long long V, int D, long long pos_rows, int dtype,
                  float scale, void* ws, size_t ws_bytes, hipStream_t s) {
    if (!em_dims(N, T, V, D, dtype) || !dtable || (dpos && pos_rows < T)) return V2A_ERR_ARG;
    if (N > 0 && (!ids || !dout)) return V2A_ERR_ARG;
#define CALL(DT)                                                                                                                                  \
    hipLaunchKernelGGL((embed_bwd_simple<DT>), dim3((unsigned)(V < 65536 ? V : 65536)), dim3(256), 0, s, ids, ids64, dout, dtable, N, V, D, scale);                          \
    if (dpos && pos_rows) hipLaunchKernelGGL((embed_dpos_kernel<DT>), dim3((unsigned)(pos_rows < 65536 ? pos_rows : 65536)), dim3(256), 0, s, ids, ids64, dout, dpos, N / T, T, V, D, pos_rows)
    EM_BY_TYPE(dtype, CALL);
#undef CALL
    V2A_CHECK_LAUNCH();
    return V2A_OK;
}

}  // extern "C"
