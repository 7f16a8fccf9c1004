// Linear attention with a decay for each head:  S_t = a_t S_{t-1} + k_t v_t^T (fp32, Dk x Dv),  a_t = exp(g_t),  o_t = scale * S_t^T q_t.
// Whole sequences (v2a_linattn_fwd / v2a_linattn_bwd) and single tokens on a pool of states (v2a_linattn_step).
#include "common.h"

namespace {

constexpr int LA_DMAX = 128;            // largest head width
constexpr float LA_GMIN = -1000.f;      // decays below exp(-1000) are 0 in fp32 already; the clamp makes -inf (a reset) ordinary arithmetic

template <int DT> struct LaT;           // element types: 0 fp32, 1 bf16, 2 fp16
template <> struct LaT<0> { typedef float T; static __device__ __forceinline__ float ld(float x) { return x; } static __device__ __forceinline__ float st(float x) { return x; } };
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

// one workgroup per (batch, head), token by token, the state in LDS
template <int DT>
__global__ __launch_bounds__(128) void la_fwd_simple(LaArgs a, void* out_, float* state_out) {
    typedef typename LaT<DT>::T E;
    __shared__ float S[LA_DMAX * LA_DMAX];
    __shared__ float qb[LA_DMAX], kb[LA_DMAX];
    const int b = blockIdx.x / a.H, h = blockIdx.x % a.H, x = threadIdx.x, Dk = a.Dk, Dv = a.Dv;
    const int hq = h / (a.H / a.Hq), hk = h / (a.H / a.Hk), hv = h / (a.H / a.Hv), n = la_len(a, b);
    const long long so = (long long)blockIdx.x * Dk * Dv;
    for (int e = x; e < Dk * Dv; e += 128) S[e] = a.state ? a.state[so + e] : 0.f;
    E* out = (E*)out_;
    for (int t = 0; t < a.T; ++t) {
        E* o = out + (((long long)b * a.T + t) * a.H + h) * Dv;
        if (t >= n) { if (x < Dv) o[x] = LaT<DT>::st(0.f); continue; }
        __syncthreads();
        if (x < Dk) {
            qb[x] = LaT<DT>::ld(((const E*)a.q)[b * a.qs[0] + t * a.qs[1] + hq * a.qs[2] + x]);
            kb[x] = LaT<DT>::ld(((const E*)a.k)[b * a.ks[0] + t * a.ks[1] + hk * a.ks[2] + x]);
        }
        __syncthreads();
        if (x < Dv) {
            const float w = expf(la_clampg(a.g[b * a.gs[0] + t * a.gs[1] + h * a.gs[2]]));
            const float vv = LaT<DT>::ld(((const E*)a.v)[b * a.vs[0] + t * a.vs[1] + hv * a.vs[2] + x]);
            float s = 0.f;
            for (int c = 0; c < Dk; ++c) {
                const float y = S[c * Dv + x] * w + kb[c] * vv;
                S[c * Dv + x] = y;
                s += qb[c] * y;
            }
            o[x] = LaT<DT>::st(s * a.scale);
        }
    }
    __syncthreads();
    if (state_out) for (int e = x; e < Dk * Dv; e += 128) state_out[so + e] = S[e];
}

// forward pass of the gradient: dq per head and the last state
template <int DT>
__global__ __launch_bounds__(128) void la_bwd_q_simple(LaArgs a, float* dqh, float* last) {
    typedef typename LaT<DT>::T E;
    __shared__ float S[LA_DMAX * LA_DMAX];
    __shared__ float kb[LA_DMAX], vb[LA_DMAX], db[LA_DMAX];
    const int b = blockIdx.x / a.H, h = blockIdx.x % a.H, x = threadIdx.x, Dk = a.Dk, Dv = a.Dv;
    const int hk = h / (a.H / a.Hk), hv = h / (a.H / a.Hv), n = la_len(a, b);
    const long long so = (long long)blockIdx.x * Dk * Dv;
    for (int e = x; e < Dk * Dv; e += 128) S[e] = a.state ? a.state[so + e] : 0.f;
    for (int t = 0; t < a.T; ++t) {
        float* o = dqh + (((long long)b * a.T + t) * a.H + h) * Dk;
        if (t >= n) { if (x < Dk) o[x] = 0.f; continue; }
        __syncthreads();
        if (x < Dk) kb[x] = LaT<DT>::ld(((const E*)a.k)[b * a.ks[0] + t * a.ks[1] + hk * a.ks[2] + x]);
        if (x < Dv) {
            vb[x] = LaT<DT>::ld(((const E*)a.v)[b * a.vs[0] + t * a.vs[1] + hv * a.vs[2] + x]);
            db[x] = LaT<DT>::ld(((const E*)a.dout)[b * a.ds[0] + t * a.ds[1] + h * a.ds[2] + x]);
        }
        __syncthreads();
        if (x < Dk) {
            const float w = expf(la_clampg(a.g[b * a.gs[0] + t * a.gs[1] + h * a.gs[2]]));
            float s = 0.f;
            for (int c = 0; c < Dv; ++c) {
                const float y = S[x * Dv + c] * w + kb[x] * vb[c];
                S[x * Dv + c] = y;
                s += db[c] * y;
            }
            o[x] = s * a.scale;
        }
    }
    __syncthreads();
    for (int e = x; e < Dk * Dv; e += 128) last[so + e] = S[e];
}

__device__ double la_blocksum(double v, double* red) {
    v = wave_sum_d(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return red[0] + red[1];
}

// reverse pass: dk, dv per head, d decay per token, gradient of the first state
template <int DT>
__global__ __launch_bounds__(128) void la_bwd_kv_simple(LaArgs a, const float* dqh, const float* last, const float* dlast, float* dkh, float* dvh,
                                                        float* dgt, float* dstate) {
    typedef typename LaT<DT>::T E;
    __shared__ float S[LA_DMAX * LA_DMAX];
    __shared__ float qb[LA_DMAX], kb[LA_DMAX], vb[LA_DMAX], db[LA_DMAX];
    __shared__ double red[2];
    const int b = blockIdx.x / a.H, h = blockIdx.x % a.H, x = threadIdx.x, Dk = a.Dk, Dv = a.Dv;
    const int hq = h / (a.H / a.Hq), hk = h / (a.H / a.Hk), hv = h / (a.H / a.Hv), n = la_len(a, b);
    const long long so = (long long)blockIdx.x * Dk * Dv;
    double cross = 0.0;
    for (int e = x; e < Dk * Dv; e += 128) {
        S[e] = dlast ? dlast[so + e] : 0.f;
        cross += (double)S[e] * last[so + e];
    }
    cross = la_blocksum(cross, red);
    for (int t = a.T - 1; t >= 0; --t) {
        const long long row = ((long long)b * a.T + t) * a.H + h;
        if (t >= n) {
            if (x < Dk) dkh[row * Dk + x] = 0.f;
            if (x < Dv) dvh[row * Dv + x] = 0.f;
            if (x == 0) dgt[row] = 0.f;
            continue;
        }
        __syncthreads();
        if (x < Dk) {
            qb[x] = LaT<DT>::ld(((const E*)a.q)[b * a.qs[0] + t * a.qs[1] + hq * a.qs[2] + x]);
            kb[x] = LaT<DT>::ld(((const E*)a.k)[b * a.ks[0] + t * a.ks[1] + hk * a.ks[2] + x]);
        }
        if (x < Dv) {
            vb[x] = LaT<DT>::ld(((const E*)a.v)[b * a.vs[0] + t * a.vs[1] + hv * a.vs[2] + x]);
            db[x] = LaT<DT>::ld(((const E*)a.dout)[b * a.ds[0] + t * a.ds[1] + h * a.ds[2] + x]) * a.scale;
        }
        __syncthreads();
        float dkx = 0.f, dvx = 0.f;
        if (x < Dk)
            for (int c = 0; c < Dv; ++c) {
                const float y = S[x * Dv + c] + qb[x] * db[c];
                S[x * Dv + c] = y;
                dkx += y * vb[c];
            }
        __syncthreads();
        if (x < Dv)
            for (int c = 0; c < Dk; ++c) dvx += S[c * Dv + x] * kb[c];
        double diff = 0.0;
        if (x < Dk) {
            dkh[row * Dk + x] = dkx;
            diff = (double)qb[x] * dqh[row * Dk + x] - (double)kb[x] * dkx;
        }
        if (x < Dv) dvh[row * Dv + x] = dvx;
        cross += la_blocksum(diff, red);
        if (x == 0) dgt[row] = (float)cross;
        const float w = expf(la_clampg(a.g[b * a.gs[0] + t * a.gs[1] + h * a.gs[2]]));
        for (int e = x; e < Dk * Dv; e += 128) S[e] *= w;
    }
    __syncthreads();
    if (dstate) for (int e = x; e < Dk * Dv; e += 128) dstate[so + e] = S[e];
}

// gradients of shared heads: the heads of a group summed in order, rounded once
template <int DT>
__global__ void la_share(const float* src, void* dst_, long long rows, int Hx, int rep, int D) {
    typedef typename LaT<DT>::T E;
    E* dst = (E*)dst_;
    const long long n = rows * Hx * D;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const long long r = i / D;
        const int c = (int)(i - r * D);
        float s = 0.f;
        for (int j = 0; j < rep; ++j) s += src[(r * rep + j) * D + c];
        dst[i] = LaT<DT>::st(s);
    }
}

// d decay of a per-head decay: the sum over all tokens, one workgroup per head, in fp64
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
// One workgroup per (row, head).  Rows that name the same slot are taken by the first of them, in row order, as successive tokens.
template <int DT>
__global__ __launch_bounds__(256) void la_step_kernel(const void* q_, const void* k_, const void* v_, const float* g, float* state, const int* slots,
                                                      void* out_, long long qb_, long long qh_, long long kb_, long long kh_, long long vb_, long long vh_,
                                                      long long gb_, long long gh_, int B, int N, int H, int Hq, int Hk, int Hv, int Dk, int Dv, float scale) {
    typedef typename LaT<DT>::T E;
    __shared__ float qs[LA_DMAX], ks[LA_DMAX];
    __shared__ float red[256];
    const int x = threadIdx.x, h = blockIdx.x % H;
    int b = blockIdx.x / H;
    int slot = b;
    E* out = (E*)out_;
    if (slots) {
        slot = slots[b];
        if (slot < 0 || slot >= N) {
            for (int c = x; c < Dv; c += 256) out[((long long)b * H + h) * Dv + c] = LaT<DT>::st(0.f);
            return;
        }
        int low = 0;
        for (int j = x; j < b; j += 256) low |= slots[j] == slot;
        if (__syncthreads_or(low)) return;
    }
    float* S = state + ((long long)slot * H + h) * Dk * Dv;
    while (b < B) {
        const E* q = (const E*)q_ + b * qb_ + (h / (H / Hq)) * qh_;
        const E* k = (const E*)k_ + b * kb_ + (h / (H / Hk)) * kh_;
        const E* v = (const E*)v_ + b * vb_ + (h / (H / Hv)) * vh_;
        const float w = expf(la_clampg(g[b * gb_ + h * gh_]));
        __syncthreads();
        if (x < Dk) { qs[x] = LaT<DT>::ld(q[x]) * scale; ks[x] = LaT<DT>::ld(k[x]); }
        __syncthreads();
        const int c = x & 127, r0 = x >> 7;
        float o = 0.f;
        if (c < Dv) {
            const float vv = LaT<DT>::ld(v[c]);
            for (int r = r0; r < Dk; r += 2) {
                const float y = S[(long long)r * Dv + c] * w + ks[r] * vv;
                S[(long long)r * Dv + c] = y;
                o += qs[r] * y;
            }
        }
        red[x] = o;
        __syncthreads();
        if (x < Dv) out[((long long)b * H + h) * Dv + x] = LaT<DT>::st(red[x] + red[x + 128]);
        if (!slots) return;
        int next = 0x7fffffff;
        for (int j = b + 1 + x; j < B; j += 256)
            if (slots[j] == slot) { next = j; break; }
        if (!__syncthreads_or(next != 0x7fffffff)) return;
        ((int*)red)[x] = next;
        __syncthreads();
        for (int j = 0; j < 256; ++j) next = min(next, ((int*)red)[j]);
        b = next;
        __syncthreads();
    }
}

bool la_dims(int B, int T, int H, int Hq, int Hk, int Hv, int Dk, int Dv, int dtype) {
    return B >= 0 && T >= 0 && H > 0 && Hq > 0 && Hk > 0 && Hv > 0 && H % Hq == 0 && H % Hk == 0 && H % Hv == 0 && Dk > 0 && Dk <= LA_DMAX && Dv > 0 &&
           Dv <= LA_DMAX && dtype >= 0 && dtype <= 2 && (long long)B * H < (1ll << 23);      // grid x block stays below 2^32 threads
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

}  // namespace

extern "C" {

size_t v2a_linattn_fwd_workspace_bytes(int B, int T, int H, int Dk, int Dv, int dtype) {
    (void)B; (void)T; (void)H; (void)Dk; (void)Dv; (void)dtype;
    return 0;
}

int v2a_linattn_fwd(const void* q, const void* k, const void* v, const float* g, const float* state, const int32_t* lens, void* out, float* state_out,
                    const int64_t* strides, int B, int T, int H, int Hq, int Hk, int Hv, int Dk, int Dv, int dtype, float scale, void* ws, size_t ws_bytes,
                    hipStream_t s) {
    if (!strides || !la_dims(B, T, H, Hq, Hk, Hv, Dk, Dv, dtype)) return V2A_ERR_ARG;
    if (B == 0 || (T == 0 && !state_out)) return V2A_OK;
    if (T > 0 && (!q || !k || !v || !g || !out)) return V2A_ERR_ARG;
    const LaArgs a = la_args(q, k, v, g, state, lens, nullptr, strides, B, T, H, Hq, Hk, Hv, Dk, Dv, scale);
#define CALL(DT) hipLaunchKernelGGL((la_fwd_simple<DT>), dim3(B * H), dim3(128), 0, s, a, out, state_out)
    LA_BY_TYPE(dtype, CALL);
#undef CALL
    V2A_CHECK_LAUNCH();
    return V2A_OK;
}

size_t v2a_linattn_bwd_workspace_bytes(int B, int T, int H, int Hq, int Hk, int Hv, int Dk, int Dv, int dtype, int per_token_decay) {
    if (!la_dims(B, T, H, Hq, Hk, Hv, Dk, Dv, dtype)) return 0;
    const size_t n = (size_t)B * T * H;
    return 2 * la_up(n * Dk * 4) + la_up(n * Dv * 4) + la_up((size_t)B * H * Dk * Dv * 4) + la_up(n * 4);
}

int v2a_linattn_bwd(const void* q, const void* k, const void* v, const float* g, const float* state, const int32_t* lens, const void* dout,
                    const float* dstate_out, void* dq, void* dk, void* dv, float* dg, float* dstate, const int64_t* strides, int B, int T, int H, int Hq, int Hk,
                    int Hv, int Dk, int Dv, int dtype, int per_token_decay, float scale, void* ws, size_t ws_bytes, hipStream_t s) {
    if (!strides || !la_dims(B, T, H, Hq, Hk, Hv, Dk, Dv, dtype)) return V2A_ERR_ARG;
    if (B > 0 && T > 0 && (!q || !k || !v || !g || !dout || !dq || !dk || !dv)) return V2A_ERR_ARG;
    if (ws_bytes < v2a_linattn_bwd_workspace_bytes(B, T, H, Hq, Hk, Hv, Dk, Dv, dtype, per_token_decay) || (ws_bytes && !ws)) return V2A_ERR_WORKSPACE;
    const LaArgs a = la_args(q, k, v, g, state, lens, dout, strides, B, T, H, Hq, Hk, Hv, Dk, Dv, scale);
    const size_t n = (size_t)B * T * H;
    char* p = (char*)ws;
    float* dqh = (float*)p; p += la_up(n * Dk * 4);
    float* dkh = (float*)p; p += la_up(n * Dk * 4);
    float* dvh = (float*)p; p += la_up(n * Dv * 4);
    float* last = (float*)p; p += la_up((size_t)B * H * Dk * Dv * 4);
    float* dgt = per_token_decay && dg ? dg : (float*)p;
    if (B > 0) {
#define CALL(DT)                                                                                        \
    hipLaunchKernelGGL((la_bwd_q_simple<DT>), dim3(B * H), dim3(128), 0, s, a, dqh, last);              \
    hipLaunchKernelGGL((la_bwd_kv_simple<DT>), dim3(B * H), dim3(128), 0, s, a, dqh, last, dstate_out, dkh, dvh, dgt, dstate)
        LA_BY_TYPE(dtype, CALL);
#undef CALL
        const long long rows = (long long)B * T;
        if (rows > 0) {
#define CALL(DT)                                                                                                                   \
    hipLaunchKernelGGL((la_share<DT>), dim3(1024), dim3(256), 0, s, dqh, dq, rows, Hq, H / Hq, Dk);                                \
    hipLaunchKernelGGL((la_share<DT>), dim3(1024), dim3(256), 0, s, dkh, dk, rows, Hk, H / Hk, Dk);                                \
    hipLaunchKernelGGL((la_share<DT>), dim3(1024), dim3(256), 0, s, dvh, dv, rows, Hv, H / Hv, Dv)
            LA_BY_TYPE(dtype, CALL);
#undef CALL
        }
    }
    if (dg && !per_token_decay) hipLaunchKernelGGL(la_dg_heads, dim3(H), dim3(256), 0, s, dgt, dg, (long long)B * T, H);
    V2A_CHECK_LAUNCH();
    return V2A_OK;
}

int v2a_linattn_step(const void* q, const void* k, const void* v, const float* g, float* state, const int32_t* slots, void* out, const int64_t* strides, int B,
                     int N, int H, int Hq, int Hk, int Hv, int Dk, int Dv, int dtype, float scale, hipStream_t s) {
    if (!strides || !la_dims(B, 1, H, Hq, Hk, Hv, Dk, Dv, dtype) || N < 0 || (!slots && N < B)) return V2A_ERR_ARG;
    if (B == 0) return V2A_OK;
    if (!q || !k || !v || !g || !state || !out) return V2A_ERR_ARG;
    const int64_t* t = strides;
#define CALL(DT)                                                                                                                                        \
    hipLaunchKernelGGL((la_step_kernel<DT>), dim3(B * H), dim3(256), 0, s, q, k, v, g, state, slots, out, (long long)t[0], (long long)t[1],              \
                       (long long)t[2], (long long)t[3], (long long)t[4], (long long)t[5], (long long)t[6], (long long)t[7], B, N, H, Hq, Hk, Hv, Dk, Dv, scale)
    LA_BY_TYPE(dtype, CALL);
#undef CALL
    V2A_CHECK_LAUNCH();
    return V2A_OK;
}

}  // extern "C"
