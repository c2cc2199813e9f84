// Group norm over channels-last activations x [N, L, C], with the activation and the dropout behind it in the same pass:
//   h = (x - mean) / sqrt(var + eps) over the L * C/G values of a sample's group,  u = gamma h + beta,  y = dropout(f(u))
// and its gradients: with du = dropout(dy) f'(u),
//   dbeta = sum du, dgamma = sum du h (over samples and positions),
//   dx = (gamma du - mean(gamma du) - h mean(gamma du h)) / sqrt(var + eps)
//
// Two passes: sums of each (sample, row range, group), then the elementwise pass, whose CTAs first add up the few sums of
// their groups.  The order of every addition is fixed by the shape alone.
//
// The forward sums are x and x^2 in 64 bits: (sum x^2) / M - mean^2 then keeps the variance of data whose mean is up to 10^6 times
// their spread, in one pass over them (activations of distance layers are all positive, far from 0 against their spread).
#include "group_norm.cuh"

namespace linf {
namespace {

// ---- forward ------------------------------------------------------------------------------------------------------

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads)
norm_sums_kernel(const T* __restrict__ x, NormDims d, NormPlan p, double2* __restrict__ part) {
    extern __shared__ double2 red[];                            // [rt][tx * V]
    const int n = blockIdx.x / p.blocks, split = blockIdx.y;
    const NormBlock b = norm_block(d, p, blockIdx.x - n * p.blocks);
    const int rt = threadIdx.x / p.tx, cv = threadIdx.x - rt * p.tx;
    double s[V], q[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = q[j] = 0.0;
    if (rt < p.rt && cv < b.nvec) {
        const int r1 = min(d.L, (split + 1) * p.rows);
        const T* at = x + ((size_t)n * d.L) * d.C + b.c0 + cv * V;
        for (int r = split * p.rows + rt; r < r1; r += 4 * p.rt) {
            Raw<T, V> v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (r + k * p.rt < r1) v[k] = load_raw<T, V>(at + (size_t)(r + k * p.rt) * d.C);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (r + k * p.rt < r1) {
                    float f[V];
                    unpack<T, V>(v[k], f);
#pragma unroll
                    for (int j = 0; j < V; ++j) { const double e = f[j]; s[j] += e; q[j] = fma(e, e, q[j]); }
                }
        }
    }
    const int width = p.tx * V;
    if (rt < p.rt) {
#pragma unroll
        for (int j = 0; j < V; ++j) red[rt * width + cv * V + j] = make_double2(s[j], q[j]);
    }
    __syncthreads();
    const int lane = threadIdx.x & 31;
    const int per = p.pieces == 1 ? d.Cg : b.nvec * V;          // channels of a group in this block
    for (int g = threadIdx.x >> 5; g < b.ng; g += kNormThreads / 32) {
        double a = 0.0, e = 0.0;
        for (int c = lane; c < per; c += 32)
            for (int r = 0; r < p.rt; ++r) {
                const double2 v = red[r * width + g * per + c];
                a += v.x;
                e += v.y;
            }
        a = warp_sum(a);
        e = warp_sum(e);
        if (lane == 0) part[(((size_t)n * p.splits + split) * d.G + b.g0 + g) * p.pieces + b.piece] = make_double2(a, e);
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads)
norm_apply_kernel(const T* __restrict__ x, const void* __restrict__ gamma, const void* __restrict__ beta, int ptype,
                  const double2* __restrict__ part, NormDims d, NormPlan p, double eps, int act, Drop drop,
                  T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
    __shared__ float2 stat[kNormMaxGroups];
    const int n = blockIdx.x / p.blocks, split = blockIdx.y;
    const NormBlock b = norm_block(d, p, blockIdx.x - n * p.blocks);
    const int lane = threadIdx.x & 31;
    for (int g = threadIdx.x >> 5; g < b.ng; g += kNormThreads / 32) {
        double a = 0.0, e = 0.0;
        for (int k = lane; k < p.splits * p.pieces; k += 32) {
            const int s = k / p.pieces, piece = k - s * p.pieces;
            const double2 v = part[(((size_t)n * p.splits + s) * d.G + b.g0 + g) * p.pieces + piece];
            a += v.x;
            e += v.y;
        }
        a = warp_sum(a) * d.inv_m;
        e = warp_sum(e) * d.inv_m - a * a;
        if (lane == 0) {
            const float m = (float)a, r = (float)(1.0 / sqrt((e > 0.0 || e != e ? e : 0.0) + eps));
            stat[g] = make_float2(m, r);
            if (split == 0 && b.piece == 0 && mean != nullptr) {
                mean[(size_t)n * d.G + b.g0 + g] = m;
                rstd[(size_t)n * d.G + b.g0 + g] = r;
            }
        }
    }
    __syncthreads();
    const int rt = threadIdx.x / p.tx, cv = threadIdx.x - rt * p.tx;
    if (rt >= p.rt || cv >= b.nvec) return;
    float m[V], r[V], w[V], o[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = cv * V + j, g = p.pieces == 1 ? c / d.Cg : 0;
        m[j] = stat[g].x;
        r[j] = stat[g].y;
        w[j] = gamma != nullptr ? load_param(gamma, b.c0 + c, ptype) : 1.f;
        o[j] = beta != nullptr ? load_param(beta, b.c0 + c, ptype) : 0.f;
    }
    DropKey key = {};
    if (drop.rng != nullptr) key = drop_key(drop);
    const int r1 = min(d.L, (split + 1) * p.rows);
    const size_t at = ((size_t)n * d.L) * d.C + b.c0 + cv * V;
    for (int l = split * p.rows + rt; l < r1; l += p.rt) {
        const size_t i = at + (size_t)l * d.C;
        float f[V];
        unpack<T, V>(load_raw<T, V>(x + i), f);
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = activate(fmaf((f[j] - m[j]) * r[j], w[j], o[j]), act);
        if (drop.rng != nullptr) drop_apply<V>(drop, key, i, f);
        store_once<T, V>(y + i, pack<T, V>(f));
    }
}

// ---- backward -----------------------------------------------------------------------------------------------------

// the gradient at u and the normalised value h of V elements
template <typename T, int V>
__device__ __forceinline__ void norm_du(const Raw<T, V>& xv, const Raw<T, V>& gv, const float (&m)[V], const float (&r)[V], const float (&w)[V],
                                        const float (&o)[V], int act, const Drop& drop, const DropKey& key, size_t i, float (&du)[V], float (&h)[V]) {
    unpack<T, V>(xv, h);
    unpack<T, V>(gv, du);
    if (drop.rng != nullptr) drop_apply<V>(drop, key, i, du);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        h[j] = (h[j] - m[j]) * r[j];
        du[j] *= slope(fmaf(h[j], w[j], o[j]), act);
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads)
norm_back_sums_kernel(const T* __restrict__ dy, const T* __restrict__ x, const void* __restrict__ gamma, const void* __restrict__ beta, int ptype,
                      const float* __restrict__ mean, const float* __restrict__ rstd, NormDims d, NormPlan p, int act, Drop drop,
                      float2* __restrict__ by_channel, float2* __restrict__ by_group) {
    extern __shared__ float2 redf[];                            // [rt][tx * V]
    const int n = blockIdx.x / p.blocks, split = blockIdx.y;
    const NormBlock b = norm_block(d, p, blockIdx.x - n * p.blocks);
    const int rt = threadIdx.x / p.tx, cv = threadIdx.x - rt * p.tx;
    const int width = p.tx * V;
    if (rt < p.rt) {
        float sa[V], sb[V];
#pragma unroll
        for (int j = 0; j < V; ++j) sa[j] = sb[j] = 0.f;
        if (cv < b.nvec) {
            float m[V], r[V], w[V], o[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int c = cv * V + j, g = b.g0 + (p.pieces == 1 ? c / d.Cg : 0);
                m[j] = mean[(size_t)n * d.G + g];
                r[j] = rstd[(size_t)n * d.G + g];
                w[j] = gamma != nullptr ? load_param(gamma, b.c0 + c, ptype) : 1.f;
                o[j] = beta != nullptr ? load_param(beta, b.c0 + c, ptype) : 0.f;
            }
            DropKey key = {};
            if (drop.rng != nullptr) key = drop_key(drop);
            const int r1 = min(d.L, (split + 1) * p.rows);
            const size_t at = ((size_t)n * d.L) * d.C + b.c0 + cv * V;
            for (int l = split * p.rows + rt; l < r1; l += p.rt) {
                const size_t i = at + (size_t)l * d.C;
                float du[V], h[V];
                norm_du<T, V>(load_raw<T, V>(x + i), load_raw<T, V>(dy + i), m, r, w, o, act, drop, key, i, du, h);
#pragma unroll
                for (int j = 0; j < V; ++j) { sa[j] += du[j]; sb[j] = fmaf(du[j], h[j], sb[j]); }
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) redf[rt * width + cv * V + j] = make_float2(sa[j], sb[j]);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < b.nvec * V; c += kNormThreads) {
        float2 t = redf[c];
        for (int k = 1; k < p.rt; ++k) { t.x += redf[k * width + c].x; t.y += redf[k * width + c].y; }
        redf[c] = t;
        by_channel[((size_t)n * p.splits + split) * d.C + b.c0 + c] = t;
    }
    __syncthreads();
    const int lane = threadIdx.x & 31;
    const int per = p.pieces == 1 ? d.Cg : b.nvec * V;
    for (int g = threadIdx.x >> 5; g < b.ng; g += kNormThreads / 32) {
        double a = 0.0, e = 0.0;
        for (int c = lane; c < per; c += 32) {
            const float w = gamma != nullptr ? load_param(gamma, b.c0 + g * per + c, ptype) : 1.f;
            a += w * redf[g * per + c].x;
            e += w * redf[g * per + c].y;
        }
        a = warp_sum(a);
        e = warp_sum(e);
        if (lane == 0) by_group[(((size_t)n * p.splits + split) * d.G + b.g0 + g) * p.pieces + b.piece] = make_float2((float)a, (float)e);
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads)
norm_back_apply_kernel(const T* __restrict__ dy, const T* __restrict__ x, const void* __restrict__ gamma, const void* __restrict__ beta, int ptype,
                       const float* __restrict__ mean, const float* __restrict__ rstd, NormDims d, NormPlan p, int act, Drop drop,
                       const float2* __restrict__ by_group, T* __restrict__ dx) {
    __shared__ float2 stat[kNormMaxGroups];
    const int n = blockIdx.x / p.blocks, split = blockIdx.y;
    const NormBlock b = norm_block(d, p, blockIdx.x - n * p.blocks);
    const int lane = threadIdx.x & 31;
    for (int g = threadIdx.x >> 5; g < b.ng; g += kNormThreads / 32) {
        double a = 0.0, e = 0.0;
        for (int k = lane; k < p.splits * p.pieces; k += 32) {
            const int s = k / p.pieces, piece = k - s * p.pieces;
            const float2 v = by_group[(((size_t)n * p.splits + s) * d.G + b.g0 + g) * p.pieces + piece];
            a += v.x;
            e += v.y;
        }
        a = warp_sum(a) * d.inv_m;
        e = warp_sum(e) * d.inv_m;
        if (lane == 0) stat[g] = make_float2((float)a, (float)e);
    }
    __syncthreads();
    const int rt = threadIdx.x / p.tx, cv = threadIdx.x - rt * p.tx;
    if (rt >= p.rt || cv >= b.nvec) return;
    float m[V], r[V], w[V], o[V], ma[V], mb[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = cv * V + j, g = p.pieces == 1 ? c / d.Cg : 0;
        m[j] = mean[(size_t)n * d.G + b.g0 + g];
        r[j] = rstd[(size_t)n * d.G + b.g0 + g];
        ma[j] = stat[g].x;
        mb[j] = stat[g].y;
        w[j] = gamma != nullptr ? load_param(gamma, b.c0 + c, ptype) : 1.f;
        o[j] = beta != nullptr ? load_param(beta, b.c0 + c, ptype) : 0.f;
    }
    DropKey key = {};
    if (drop.rng != nullptr) key = drop_key(drop);
    const int r1 = min(d.L, (split + 1) * p.rows);
    const size_t at = ((size_t)n * d.L) * d.C + b.c0 + cv * V;
    for (int l = split * p.rows + rt; l < r1; l += p.rt) {
        const size_t i = at + (size_t)l * d.C;
        float du[V], h[V];
        norm_du<T, V>(load_raw<T, V>(x + i), load_raw<T, V>(dy + i), m, r, w, o, act, drop, key, i, du, h);
#pragma unroll
        for (int j = 0; j < V; ++j) du[j] = r[j] * (fmaf(w[j], du[j], -ma[j]) - h[j] * mb[j]);
        store_once<T, V>(dx + i, pack<T, V>(du));
    }
}

// dgamma, dbeta: the per-channel sums of all samples and row ranges, in 64 bits, 32 channels to a CTA
__global__ void __launch_bounds__(1024)
norm_params_kernel(const float2* __restrict__ by_channel, long long count, int C, void* __restrict__ dgamma, void* __restrict__ dbeta, int ptype) {
    __shared__ double red[2][32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    double a = 0.0, e = 0.0;
    if (c < C)
        for (long long k = warp; k < count; k += 32) {
            const float2 v = __ldg(by_channel + k * C + c);
            a += v.x;
            e += v.y;
        }
    red[0][warp][lane] = a;
    red[1][warp][lane] = e;
    __syncthreads();
    a = warp_sum(red[0][lane][warp]);
    e = warp_sum(red[1][lane][warp]);
    const int out = blockIdx.x * 32 + warp;
    if (lane == 0 && out < C) {
        if (dbeta != nullptr) store_param(dbeta, out, ptype, (float)a);
        if (dgamma != nullptr) store_param(dgamma, out, ptype, (float)e);
    }
}

template <typename T, int V>
int forward(const T* x, const void* gamma, const void* beta, int ptype, const NormDims& d, const NormPlan& p, double eps, int act,
            const Drop& drop, T* y, float* mean, float* rstd, void* ws, cudaStream_t st) {
    const dim3 grid((unsigned)(p.blocks * d.N), p.splits);
    double2* part = static_cast<double2*>(ws);
    norm_sums_kernel<T, V><<<grid, kNormThreads, sizeof(double2) * p.rt * p.tx * V, st>>>(x, d, p, part);
    norm_apply_kernel<T, V><<<grid, kNormThreads, 0, st>>>(x, gamma, beta, ptype, part, d, p, eps, act, drop, y, mean, rstd);
    return launch_status(2);
}

template <typename T, int V>
int backward(const T* dy, const T* x, const void* gamma, const void* beta, int ptype, const float* mean, const float* rstd, const NormDims& d,
             const NormPlan& p, int act, const Drop& drop, T* dx, void* dgamma, void* dbeta, void* ws, cudaStream_t st) {
    const dim3 grid((unsigned)(p.blocks * d.N), p.splits);
    float2* by_channel = static_cast<float2*>(ws);
    float2* by_group = by_channel + (size_t)d.N * p.splits * d.C;
    int launched = 1;
    norm_back_sums_kernel<T, V><<<grid, kNormThreads, sizeof(float2) * p.rt * p.tx * V, st>>>(dy, x, gamma, beta, ptype, mean, rstd, d, p, act,
                                                                                                 drop, by_channel, by_group);
    if (dx != nullptr) {
        norm_back_apply_kernel<T, V><<<grid, kNormThreads, 0, st>>>(dy, x, gamma, beta, ptype, mean, rstd, d, p, act, drop, by_group, dx);
        ++launched;
    }
    if (launch_status(launched)) return LINF_ERR_LAUNCH;
    return dgamma != nullptr || dbeta != nullptr ? norm_params(by_channel, (long long)d.N * p.splits, d.C, dgamma, dbeta, ptype, st) : LINF_OK;
}

size_t workspace(const NormDims& d, const NormPlan& p, bool back) {
    const size_t groups = (size_t)d.N * p.splits * d.G * p.pieces;
    return back ? sizeof(float2) * ((size_t)d.N * p.splits * d.C + groups) : sizeof(double2) * groups;
}

}  // namespace

int norm_params(const float2* by_channel, long long count, int C, void* dgamma, void* dbeta, int ptype, cudaStream_t st) {
    norm_params_kernel<<<(C + 31) / 32, 1024, 0, st>>>(by_channel, count, C, dgamma, dbeta, ptype);
    return launch_status();
}

size_t group_norm_workspace(int N, int C, int G, int L, int type, bool back) {
    // a plan goes by the pointers' alignment; either may run
    size_t most = 0;
    for (int k = 0; k < 2; ++k) {
        NormDims d;
        NormPlan p;
        if (norm_make(N, C, G, L, type == LINF_F32 ? 4 : 2, k == 0, &d, &p) != LINF_OK) return 0;
        const size_t need = workspace(d, p, back);
        if (need > most) most = need;
    }
    return (most + 255) / 256 * 256;
}

#define LINF_BY_VECTOR(CALL16, CALL32)                                                                             \
    switch (type) {                                                                                                \
        case LINF_F32:                                                                                             \
            if (p.V == 4) return CALL32(float, 4);                                                                 \
            return CALL32(float, 1);                                                                               \
        case LINF_F16:                                                                                             \
            if (p.V == 8) return CALL16(__half, 8);                                                                \
            if (p.V == 2) return CALL16(__half, 2);                                                                \
            return CALL16(__half, 1);                                                                              \
        default:                                                                                                   \
            if (p.V == 8) return CALL16(__nv_bfloat16, 8);                                                         \
            if (p.V == 2) return CALL16(__nv_bfloat16, 2);                                                         \
            return CALL16(__nv_bfloat16, 1);                                                                       \
    }

int group_norm_forward(const void* x, const void* gamma, const void* beta, int N, int C, int G, int L, int type, int ptype, double eps, int act,
                       double rate, const long long* rng, void* y, float* mean, float* rstd, void* ws, size_t ws_bytes, cudaStream_t st) {
    NormDims d;
    NormPlan p;
    Drop drop;
    if (!make_drop(rate, rng, &drop)) return LINF_ERR_RATE;
    const int rc = norm_make(N, C, G, L, type == LINF_F32 ? 4 : 2, aligned16(x) && aligned16(y), &d, &p);
    if (rc) return rc;
    if (ws == nullptr || !aligned16(ws) || ws_bytes < workspace(d, p, false)) return LINF_ERR_WORKSPACE;
#define LINF_CALL(T, V) forward<T, V>(static_cast<const T*>(x), gamma, beta, ptype, d, p, eps, act, drop, static_cast<T*>(y), mean, rstd, ws, st)
    LINF_BY_VECTOR(LINF_CALL, LINF_CALL)
#undef LINF_CALL
}

int group_norm_backward(const void* dy, const void* x, const void* gamma, const void* beta, const float* mean, const float* rstd, int N, int C,
                        int G, int L, int type, int ptype, int act, double rate, const long long* rng, void* dx, void* dgamma, void* dbeta,
                        void* ws, size_t ws_bytes, cudaStream_t st) {
    NormDims d;
    NormPlan p;
    Drop drop;
    if (!make_drop(rate, rng, &drop)) return LINF_ERR_RATE;
    const int rc = norm_make(N, C, G, L, type == LINF_F32 ? 4 : 2, aligned16(x) && aligned16(dy) && aligned16(dx), &d, &p);
    if (rc) return rc;
    if (ws == nullptr || !aligned16(ws) || ws_bytes < workspace(d, p, true)) return LINF_ERR_WORKSPACE;
#define LINF_CALL(T, V)                                                                                                                   \
    backward<T, V>(static_cast<const T*>(dy), static_cast<const T*>(x), gamma, beta, ptype, mean, rstd, d, p, act, drop, static_cast<T*>(dx), \
                   dgamma, dbeta, ws, st)
    LINF_BY_VECTOR(LINF_CALL, LINF_CALL)
#undef LINF_CALL
}

}  // namespace linf
