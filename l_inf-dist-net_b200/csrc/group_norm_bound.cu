// Group norm over a box: bounds of f(gamma h(x) + beta) for every x with lower <= x <= upper, and their gradients.
//
// With L, U the sums of a group's lower and upper ends, M its size, c = (l + u) / 2 and r = (u - l) / 2:
//   x_i - mean(x) lies in [n-, n+],  n- = l - U/M + (u - l)/M,  n+ = u - L/M - (u - l)/M   (exact: x_i counts in its own mean)
//   std(x) lies in [max(0, std(c) - rho), std(c) + rho],  rho = sqrt(mean r^2)             (triangle inequality; centring never lengthens)
// so 1 / sqrt(var + eps) lies in [s_lo, s_hi], and the quotient's ends are products of ends:
//   z- = min(n- s_lo, n- s_hi),  z+ = max(n+ s_lo, n+ s_hi), cut at -+sqrt(M - 1), beyond which no normalised value of M can be.
// gamma < 0 exchanges the ends.  The activations are monotone, but for silu, which has one minimum.
//
// All of it is computed in 64 bits and rounded once: which of two ends a bound takes, and with it a gradient, is decided next to 0.
// The kernels are bound by HBM all the same (16 bytes of a forward pass stand against some 25 operations in 64 bits, and an SM issues 64 a clock).
#include "group_norm.cuh"

namespace linf {
namespace {

struct Sum4 { double a, b, c, d; };
__device__ __forceinline__ Sum4 add4(const Sum4& p, const Sum4& q) { return Sum4{p.a + q.a, p.b + q.b, p.c + q.c, p.d + q.d}; }
__device__ __forceinline__ Sum4 warp_sum4(Sum4 v) { return Sum4{warp_sum(v.a), warp_sum(v.b), warp_sum(v.c), warp_sum(v.d)}; }

// What the elements of a group share.
struct Box {
    double mean_l, mean_u, sd, rho;     // the means of the ends, std of the centres, root mean square of the radii
    double s_lo, s_hi, cut;             // range of 1 / sqrt(var + eps); sqrt(M - 1)
};

__device__ __forceinline__ Box make_box(const Sum4& s, const NormDims& d, double eps) {
    Box b;
    b.mean_l = s.a * d.inv_m;
    b.mean_u = s.b * d.inv_m;
    const double mc = (b.mean_l + b.mean_u) * 0.5, vc = 0.25 * s.c * d.inv_m - mc * mc, vr = 0.25 * s.d * d.inv_m;
    b.sd = sqrt(vc > 0.0 || vc != vc ? vc : 0.0);
    b.rho = sqrt(vr);
    const double far = b.sd + b.rho, near = fmax(b.sd - b.rho, 0.0) + (b.sd - b.rho) * 0.0;     // keeps a NaN
    b.s_lo = 1.0 / sqrt(far * far + eps);
    b.s_hi = 1.0 / sqrt(near * near + eps);
    const double m = (double)d.L * d.Cg;
    b.cut = sqrt(m - 1.0);
    return b;
}

// The range [n-, n+] of x_i - mean(x), and what it becomes.
struct Ends { double n0, n1, s0, s1, z0, z1; bool cut0, cut1; };
__device__ __forceinline__ Ends make_ends(const Box& b, double l, double u, double inv_m) {
    Ends e;
    const double own = (u - l) * inv_m;
    e.n0 = l - b.mean_u + own;
    e.n1 = u - b.mean_l - own;
    e.s0 = e.n0 >= 0.0 ? b.s_lo : b.s_hi;
    e.s1 = e.n1 >= 0.0 ? b.s_hi : b.s_lo;
    e.z0 = e.n0 * e.s0;
    e.z1 = e.n1 * e.s1;
    e.cut0 = e.z0 <= -b.cut;
    e.cut1 = e.z1 >= b.cut;
    if (e.cut0) e.z0 = -b.cut;
    if (e.cut1) e.z1 = b.cut;
    return e;
}

// Over [v0, v1] silu is largest at one of the ends, and least at one of them or at its minimum between them.  Which end, where the
// minimum lies between them, is decided in 64 bits: the two values may be equal to the last bits of fp32 while their slopes differ.
struct Sides { bool inside, top_is_v1; };
__device__ __forceinline__ Sides silu_sides(double v0, double v1) {
    Sides s;
    s.inside = v0 < kSiluArg64 && v1 > kSiluArg64;
    s.top_is_v1 = s.inside ? v1 / (1.0 + exp(-v1)) > v0 / (1.0 + exp(-v0)) : v0 >= kSiluArg64;
    return s;
}

// bounds of f over [v0, v1]
__device__ __forceinline__ void bound_act(double v0, double v1, int act, float& y0, float& y1) {
    y0 = activate((float)v0, act);
    y1 = activate((float)v1, act);
    if (act == LINF_ACT_SILU && v0 == v0 && v1 == v1) {
        const Sides s = silu_sides(v0, v1);
        const float low = s.inside ? activate(kSiluArg, act) : s.top_is_v1 ? y0 : y1, high = s.top_is_v1 ? y1 : y0;
        y0 = fminf(low, high);                      // one rounding of a flat stretch may turn two values around
        y1 = high;
    }
}
// gradients (g0, g1) at the bounds -> at v0 and v1
__device__ __forceinline__ void bound_slope(double v0, double v1, int act, float g0, float g1, double& d0, double& d1) {
    if (act == LINF_ACT_SILU) {
        const Sides s = silu_sides(v0, v1);
        const float low = s.inside ? 0.f : g0;
        const float at0 = s.top_is_v1 ? low : g1, at1 = s.top_is_v1 ? g1 : low;
        g0 = at0;
        g1 = at1;
    }
    d0 = (double)(g0 * slope((float)v0, act));
    d1 = (double)(g1 * slope((float)v1, act));
}

// adds up a CTA's per-thread values [rt][tx * V] of a group: lanes along the channels, rows in order
template <int V>
__device__ __forceinline__ Sum4 group_sum(const Sum4* red, const NormPlan& p, int per, int g) {
    Sum4 t = {0.0, 0.0, 0.0, 0.0};
    for (int c = threadIdx.x & 31; c < per; c += 32)
        for (int r = 0; r < p.rt; ++r) t = add4(t, red[r * p.tx * V + g * per + c]);
    return warp_sum4(t);
}

template <int V>
__global__ void __launch_bounds__(kNormThreads)
bound_sums_kernel(const float* __restrict__ lower, const float* __restrict__ upper, NormDims d, NormPlan p, Sum4* __restrict__ part) {
    extern __shared__ Sum4 red[];
    const int n = blockIdx.x / p.blocks, split = blockIdx.y;
    const NormBlock b = norm_block(d, p, blockIdx.x - n * p.blocks);
    const int rt = threadIdx.x / p.tx, cv = threadIdx.x - rt * p.tx;
    Sum4 s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = Sum4{0.0, 0.0, 0.0, 0.0};
    if (rt < p.rt && cv < b.nvec) {
        const int r1 = min(d.L, (split + 1) * p.rows);
        const size_t at = ((size_t)n * d.L) * d.C + b.c0 + cv * V;
#pragma unroll 2
        for (int r = split * p.rows + rt; r < r1; r += p.rt) {
            float l[V], u[V];
            unpack<float, V>(load_raw<float, V>(lower + at + (size_t)r * d.C), l);
            unpack<float, V>(load_raw<float, V>(upper + at + (size_t)r * d.C), u);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const double a = l[j], e = u[j];
                s[j].a += a;
                s[j].b += e;
                s[j].c = fma(a + e, a + e, s[j].c);
                s[j].d = fma(e - a, e - a, s[j].d);
            }
        }
    }
    if (rt < p.rt) {
#pragma unroll
        for (int j = 0; j < V; ++j) red[rt * p.tx * V + cv * V + j] = s[j];
    }
    __syncthreads();
    const int per = p.pieces == 1 ? d.Cg : b.nvec * V;
    for (int g = threadIdx.x >> 5; g < b.ng; g += kNormThreads / 32) {
        const Sum4 t = group_sum<V>(red, p, per, g);
        if ((threadIdx.x & 31) == 0) part[(((size_t)n * p.splits + split) * d.G + b.g0 + g) * p.pieces + b.piece] = t;
    }
}

// sums of a group over its row ranges and pieces
__device__ __forceinline__ Sum4 all_parts(const Sum4* part, const NormDims& d, const NormPlan& p, int n, int g) {
    Sum4 t = {0.0, 0.0, 0.0, 0.0};
    for (int k = threadIdx.x & 31; k < p.splits * p.pieces; k += 32) {
        const int s = k / p.pieces, piece = k - s * p.pieces;
        t = add4(t, part[(((size_t)n * p.splits + s) * d.G + g) * p.pieces + piece]);
    }
    return warp_sum4(t);
}

template <int V>
__global__ void __launch_bounds__(kNormThreads)
bound_apply_kernel(const float* __restrict__ lower, const float* __restrict__ upper, const float* __restrict__ gamma, const float* __restrict__ beta,
                   const Sum4* __restrict__ part, NormDims d, NormPlan p, double eps, int act, float* __restrict__ out_l, float* __restrict__ out_u,
                   Sum4* __restrict__ sums) {
    extern __shared__ Box box[];                                // [groups of the block]
    const int n = blockIdx.x / p.blocks, split = blockIdx.y;
    const NormBlock b = norm_block(d, p, blockIdx.x - n * p.blocks);
    for (int g = threadIdx.x >> 5; g < b.ng; g += kNormThreads / 32) {
        const Sum4 t = all_parts(part, d, p, n, b.g0 + g);
        if ((threadIdx.x & 31) == 0) {
            box[g] = make_box(t, d, eps);
            if (split == 0 && b.piece == 0 && sums != nullptr) sums[(size_t)n * d.G + b.g0 + g] = t;
        }
    }
    __syncthreads();
    const int rt = threadIdx.x / p.tx, cv = threadIdx.x - rt * p.tx;
    if (rt >= p.rt || cv >= b.nvec) return;
    float w[V], o[V];
    const Box* bx[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = cv * V + j;
        bx[j] = box + (p.pieces == 1 ? c / d.Cg : 0);
        w[j] = gamma != nullptr ? __ldg(gamma + b.c0 + c) : 1.f;
        o[j] = beta != nullptr ? __ldg(beta + b.c0 + c) : 0.f;
    }
    const int r1 = min(d.L, (split + 1) * p.rows);
    const size_t at = ((size_t)n * d.L) * d.C + b.c0 + cv * V;
    for (int r = split * p.rows + rt; r < r1; r += p.rt) {
        const size_t i = at + (size_t)r * d.C;
        float l[V], u[V];
        unpack<float, V>(load_raw<float, V>(lower + i), l);
        unpack<float, V>(load_raw<float, V>(upper + i), u);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const Ends e = make_ends(*bx[j], l[j], u[j], d.inv_m);
            const double z0 = w[j] < 0.f ? e.z1 : e.z0, z1 = w[j] < 0.f ? e.z0 : e.z1;
            bound_act(fma(z0, (double)w[j], (double)o[j]), fma(z1, (double)w[j], (double)o[j]), act, l[j], u[j]);
        }
        store_once<float, V>(out_l + i, pack<float, V>(l));
        store_once<float, V>(out_u + i, pack<float, V>(u));
    }
}

// gradients at z- and z+ of one element, and what they add to those of gamma and beta
__device__ __forceinline__ void bound_dz(const Ends& e, float w, float o, int act, float g0, float g1, double& q0, double& q1, double& dw, double& db) {
    const bool turned = w < 0.f;
    const double z0 = turned ? e.z1 : e.z0, z1 = turned ? e.z0 : e.z1;
    double d0, d1;
    bound_slope(fma(z0, (double)w, (double)o), fma(z1, (double)w, (double)o), act, g0, g1, d0, d1);
    dw = d0 * z0 + d1 * z1;
    db = d0 + d1;
    q0 = e.cut0 ? 0.0 : (turned ? d1 : d0) * (double)w;
    q1 = e.cut1 ? 0.0 : (turned ? d0 : d1) * (double)w;
}

template <int V>
__global__ void __launch_bounds__(kNormThreads)
bound_back_sums_kernel(const float* __restrict__ g_l, const float* __restrict__ g_u, const float* __restrict__ lower, const float* __restrict__ upper,
                       const float* __restrict__ gamma, const float* __restrict__ beta, const Sum4* __restrict__ sums, NormDims d, NormPlan p,
                       double eps, int act, float2* __restrict__ by_channel, Sum4* __restrict__ by_group) {
    extern __shared__ Sum4 red[];                               // [rt][tx * V], then the boxes
    Box* box = reinterpret_cast<Box*>(red + p.rt * p.tx * V);
    const int n = blockIdx.x / p.blocks, split = blockIdx.y;
    const NormBlock b = norm_block(d, p, blockIdx.x - n * p.blocks);
    for (int g = threadIdx.x; g < b.ng; g += kNormThreads) box[g] = make_box(sums[(size_t)n * d.G + b.g0 + g], d, eps);
    __syncthreads();
    const int rt = threadIdx.x / p.tx, cv = threadIdx.x - rt * p.tx;
    const int width = p.tx * V;
    double sw[V], sb[V];
    Sum4 s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) { s[j] = Sum4{0.0, 0.0, 0.0, 0.0}; sw[j] = sb[j] = 0.0; }
    if (rt < p.rt && cv < b.nvec) {
        float w[V], o[V];
        const Box* bx[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = cv * V + j;
            bx[j] = box + (p.pieces == 1 ? c / d.Cg : 0);
            w[j] = gamma != nullptr ? __ldg(gamma + b.c0 + c) : 1.f;
            o[j] = beta != nullptr ? __ldg(beta + b.c0 + c) : 0.f;
        }
        const int r1 = min(d.L, (split + 1) * p.rows);
        const size_t at = ((size_t)n * d.L) * d.C + b.c0 + cv * V;
        for (int r = split * p.rows + rt; r < r1; r += p.rt) {
            const size_t i = at + (size_t)r * d.C;
            float l[V], u[V], gl[V], gu[V];
            unpack<float, V>(load_raw<float, V>(lower + i), l);
            unpack<float, V>(load_raw<float, V>(upper + i), u);
            unpack<float, V>(load_raw<float, V>(g_l + i), gl);
            unpack<float, V>(load_raw<float, V>(g_u + i), gu);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const Ends e = make_ends(*bx[j], l[j], u[j], d.inv_m);
                double q0, q1, dw, db;
                bound_dz(e, w[j], o[j], act, gl[j], gu[j], q0, q1, dw, db);
                sw[j] += dw;
                sb[j] += db;
                s[j].a = fma(q0, e.s0, s[j].a);                 // the gradients at n- and n+
                s[j].b = fma(q1, e.s1, s[j].b);
                const double t0 = q0 * e.n0, t1 = q1 * e.n1;    // at s_lo and s_hi
                s[j].c += (e.n0 >= 0.0 ? t0 : 0.0) + (e.n1 >= 0.0 ? 0.0 : t1);
                s[j].d += (e.n0 >= 0.0 ? 0.0 : t0) + (e.n1 >= 0.0 ? t1 : 0.0);
            }
        }
    }
    // the channels' sums first, in the same memory
    double2* red2 = reinterpret_cast<double2*>(red);
    if (rt < p.rt) {
#pragma unroll
        for (int j = 0; j < V; ++j) red2[rt * width + cv * V + j] = make_double2(sb[j], sw[j]);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < b.nvec * V; c += kNormThreads) {
        double2 t = red2[c];
        for (int k = 1; k < p.rt; ++k) { t.x += red2[k * width + c].x; t.y += red2[k * width + c].y; }
        by_channel[((size_t)n * p.splits + split) * d.C + b.c0 + c] = make_float2((float)t.x, (float)t.y);
    }
    __syncthreads();
    if (rt < p.rt) {
#pragma unroll
        for (int j = 0; j < V; ++j) red[rt * width + cv * V + j] = s[j];
    }
    __syncthreads();
    const int per = p.pieces == 1 ? d.Cg : b.nvec * V;
    for (int g = threadIdx.x >> 5; g < b.ng; g += kNormThreads / 32) {
        const Sum4 t = group_sum<V>(red, p, per, g);
        if ((threadIdx.x & 31) == 0) by_group[(((size_t)n * p.splits + split) * d.G + b.g0 + g) * p.pieces + b.piece] = t;
    }
}

// What the elements of a group share in the backward pass.
struct Back {
    Box box;
    double s0, s1;              // means of the gradients at n- and n+
    double by_c, by_r;          // factor of c - mean(c), and of r
};

template <int V>
__global__ void __launch_bounds__(kNormThreads)
bound_back_apply_kernel(const float* __restrict__ g_l, const float* __restrict__ g_u, const float* __restrict__ lower, const float* __restrict__ upper,
                        const float* __restrict__ gamma, const float* __restrict__ beta, const Sum4* __restrict__ sums,
                        const Sum4* __restrict__ by_group, NormDims d, NormPlan p, double eps, int act, float* __restrict__ d_l, float* __restrict__ d_u) {
    extern __shared__ Back back[];
    const int n = blockIdx.x / p.blocks, split = blockIdx.y;
    const NormBlock b = norm_block(d, p, blockIdx.x - n * p.blocks);
    for (int g = threadIdx.x >> 5; g < b.ng; g += kNormThreads / 32) {
        const Sum4 t = all_parts(by_group, d, p, n, b.g0 + g);
        if ((threadIdx.x & 31) == 0) {
            Back k;
            k.box = make_box(sums[(size_t)n * d.G + b.g0 + g], d, eps);
            const Box& x = k.box;
            k.s0 = t.a * d.inv_m;
            k.s1 = t.b * d.inv_m;
            const double lo = t.c * x.s_lo * x.s_lo * x.s_lo * (x.sd + x.rho), hi = t.d * x.s_hi * x.s_hi * x.s_hi * fmax(x.sd - x.rho, 0.0);
            // std and rho have no slope at 0, where all centres are one or all radii are 0: none is passed on
            k.by_c = x.sd > 0.0 ? -(lo + hi) * d.inv_m / x.sd : 0.0;
            k.by_r = x.rho > 0.0 ? (hi - lo) * d.inv_m / x.rho : 0.0;
            back[g] = k;
        }
    }
    __syncthreads();
    const int rt = threadIdx.x / p.tx, cv = threadIdx.x - rt * p.tx;
    if (rt >= p.rt || cv >= b.nvec) return;
    float w[V], o[V];
    const Back* bk[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = cv * V + j;
        bk[j] = back + (p.pieces == 1 ? c / d.Cg : 0);
        w[j] = gamma != nullptr ? __ldg(gamma + b.c0 + c) : 1.f;
        o[j] = beta != nullptr ? __ldg(beta + b.c0 + c) : 0.f;
    }
    const int r1 = min(d.L, (split + 1) * p.rows);
    const size_t at = ((size_t)n * d.L) * d.C + b.c0 + cv * V;
    for (int r = split * p.rows + rt; r < r1; r += p.rt) {
        const size_t i = at + (size_t)r * d.C;
        float l[V], u[V], gl[V], gu[V];
        unpack<float, V>(load_raw<float, V>(lower + i), l);
        unpack<float, V>(load_raw<float, V>(upper + i), u);
        unpack<float, V>(load_raw<float, V>(g_l + i), gl);
        unpack<float, V>(load_raw<float, V>(g_u + i), gu);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const Back& k = *bk[j];
            const double a = l[j], e = u[j];
            const Ends s = make_ends(k.box, a, e, d.inv_m);
            double q0, q1, dw, db;
            bound_dz(s, w[j], o[j], act, gl[j], gu[j], q0, q1, dw, db);
            q0 *= s.s0;
            q1 *= s.s1;
            const double dc = k.by_c * ((a + e) * 0.5 - (k.box.mean_l + k.box.mean_u) * 0.5), dr = k.by_r * (e - a) * 0.5;
            gl[j] = (float)(q0 - q0 * d.inv_m + q1 * d.inv_m - k.s1 + (dc - dr) * 0.5);
            gu[j] = (float)(q1 - q1 * d.inv_m + q0 * d.inv_m - k.s0 + (dc + dr) * 0.5);
        }
        store_once<float, V>(d_l + i, pack<float, V>(gl));
        store_once<float, V>(d_u + i, pack<float, V>(gu));
    }
}

template <int V>
int forward(const float* lower, const float* upper, const float* gamma, const float* beta, const NormDims& d, const NormPlan& p, double eps, int act,
            float* out_l, float* out_u, Sum4* sums, void* ws, cudaStream_t st) {
    const dim3 grid((unsigned)(p.blocks * d.N), p.splits);
    Sum4* part = static_cast<Sum4*>(ws);
    bound_sums_kernel<V><<<grid, kNormThreads, sizeof(Sum4) * p.rt * p.tx * V, st>>>(lower, upper, d, p, part);
    const size_t boxes = sizeof(Box) * p.groups;
    if (boxes > 48 * 1024 && cudaFuncSetAttribute(bound_apply_kernel<V>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)boxes) != cudaSuccess)
        return LINF_ERR_LAUNCH;
    bound_apply_kernel<V><<<grid, kNormThreads, boxes, st>>>(lower, upper, gamma, beta, part, d, p, eps, act, out_l, out_u, sums);
    return launch_status(2);
}

template <int V>
int backward(const float* g_l, const float* g_u, const float* lower, const float* upper, const float* gamma, const float* beta, const Sum4* sums,
             const NormDims& d, const NormPlan& p, double eps, int act, float* d_l, float* d_u, float* dgamma, float* dbeta, void* ws, cudaStream_t st) {
    const dim3 grid((unsigned)(p.blocks * d.N), p.splits);
    Sum4* by_group = static_cast<Sum4*>(ws);
    float2* by_channel = reinterpret_cast<float2*>(by_group + (size_t)d.N * p.splits * d.G * p.pieces);
    const size_t one = sizeof(Sum4) * p.rt * p.tx * V + sizeof(Box) * p.groups, two = sizeof(Back) * p.groups;
    if ((one > 48 * 1024 && cudaFuncSetAttribute(bound_back_sums_kernel<V>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)one) != cudaSuccess) ||
        (two > 48 * 1024 && cudaFuncSetAttribute(bound_back_apply_kernel<V>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)two) != cudaSuccess))
        return LINF_ERR_LAUNCH;
    int launched = 1;
    bound_back_sums_kernel<V><<<grid, kNormThreads, one, st>>>(g_l, g_u, lower, upper, gamma, beta, sums, d, p, eps, act, by_channel, by_group);
    if (d_l != nullptr) {
        bound_back_apply_kernel<V><<<grid, kNormThreads, two, st>>>(g_l, g_u, lower, upper, gamma, beta, sums, by_group, d, p, eps, act, d_l, d_u);
        ++launched;
    }
    if (launch_status(launched)) return LINF_ERR_LAUNCH;
    return dgamma != nullptr || dbeta != nullptr ? norm_params(by_channel, (long long)d.N * p.splits, d.C, dgamma, dbeta, LINF_F32, st) : LINF_OK;
}

size_t workspace(const NormDims& d, const NormPlan& p, bool back) {
    return sizeof(Sum4) * (size_t)d.N * p.splits * d.G * p.pieces + (back ? sizeof(float2) * (size_t)d.N * p.splits * d.C : 0);
}

}  // namespace

size_t group_norm_bound_workspace(int N, int C, int G, int L, bool back) {
    size_t most = 0;
    for (int k = 0; k < 2; ++k) {
        NormDims d;
        NormPlan p;
        if (norm_make(N, C, G, L, 4, k == 0, &d, &p) != LINF_OK) return 0;
        const size_t need = workspace(d, p, back);
        if (need > most) most = need;
    }
    return (most + 255) / 256 * 256;
}

int group_norm_bound_forward(const float* lower, const float* upper, const float* gamma, const float* beta, int N, int C, int G, int L, double eps,
                             int act, float* out_l, float* out_u, double* sums, void* ws, size_t ws_bytes, cudaStream_t st) {
    NormDims d;
    NormPlan p;
    const int rc = norm_make(N, C, G, L, 4, aligned16(lower) && aligned16(upper) && aligned16(out_l) && aligned16(out_u), &d, &p);
    if (rc) return rc;
    if (ws == nullptr || !aligned16(ws) || ws_bytes < workspace(d, p, false)) return LINF_ERR_WORKSPACE;
    Sum4* s = reinterpret_cast<Sum4*>(sums);
    return p.V == 4 ? forward<4>(lower, upper, gamma, beta, d, p, eps, act, out_l, out_u, s, ws, st)
                    : forward<1>(lower, upper, gamma, beta, d, p, eps, act, out_l, out_u, s, ws, st);
}

int group_norm_bound_backward(const float* g_l, const float* g_u, const float* lower, const float* upper, const float* gamma, const float* beta,
                              const double* sums, int N, int C, int G, int L, double eps, int act, float* d_l, float* d_u, float* dgamma,
                              float* dbeta, void* ws, size_t ws_bytes, cudaStream_t st) {
    NormDims d;
    NormPlan p;
    const int rc = norm_make(N, C, G, L, 4, aligned16(g_l) && aligned16(g_u) && aligned16(lower) && aligned16(upper) && aligned16(d_l) && aligned16(d_u), &d, &p);
    if (rc) return rc;
    if (ws == nullptr || !aligned16(ws) || ws_bytes < workspace(d, p, true)) return LINF_ERR_WORKSPACE;
    const Sum4* s = reinterpret_cast<const Sum4*>(sums);
    return p.V == 4 ? backward<4>(g_l, g_u, lower, upper, gamma, beta, s, d, p, eps, act, d_l, d_u, dgamma, dbeta, ws, st)
                    : backward<1>(g_l, g_u, lower, upper, gamma, beta, s, d, p, eps, act, d_l, d_u, dgamma, dbeta, ws, st);
}

}  // namespace linf
