// Group norm over a box: bounds of f(gamma h(x) + beta) for every x with lower <= x <= upper, and their gradients.
//
// With L, U the sums of a group's lower and upper ends, M its size, c = (l + u) / 2 and r = (u - l) / 2:
//   x_i - mean(x) lies in [n-, n+],  n- = l - U/M + (u - l)/M,  n+ = u - L/M - (u - l)/M   (exact: x_i counts in its own mean)
//   std(x) lies in [max(0, std(c) - rho), std(c) + rho],  rho = sqrt(mean r^2)             (triangle inequality; centring never lengthens)
// so 1 / sqrt(var + eps) lies in [s_lo, s_hi], and the quotient's ends are products of ends:
//   z- = min(n- s_lo, n- s_hi),  z+ = max(n+ s_lo, n+ s_hi), cut at -+sqrt(M - 1), beyond which no normalised value of M can be.
// gamma < 0 exchanges the ends.  The activations are monotone, but for silu, which has one minimum.
//
// Sums, and all of the backward pass, are computed in 64 bits: which of two ends a bound takes, and with it a gradient, is decided next to
// 0.  The elements of the forward pass, whose values do not jump there, are fp32, with the means in two parts, so that no bound is off by more
// than a few roundings of its own terms.  Of the backward pass the activation's slope and its product with a gradient are fp32, and so are the
// partial sums for gamma and beta that a CTA leaves behind.
//
// What bounds it: latency.  Forward passes over maps are at half of HBM's peak with 19 to 22 warps on an SM; the backward passes, with 14 to 15 warps,
// 94 to 128 registers and loads that go straight to registers, at a quarter of it, and at a quarter of the 64-bit units' rate.  Measured on one B200,
// us: 32 x 192 x 56 x 56, relu, forward 96 (elements in 64 bits: 119; 47 if all crossed HBM once); 16 x 192 x 56 x 56, tanh, both directions 236;
// 512 x 512, 16 groups, tanh, both 25.
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

// One value of each group of sample n from group g0 on, each d.Cg apart (the first lower end of a row in the middle).  The squares of the centres are
// taken about it: boxes far from 0 against their spread would lose the spread in the difference of two large sums.
__device__ __forceinline__ const float* level_of(const float* lower, const NormDims& d, int n, int g0) {
    return lower + ((size_t)n * d.L + d.L / 2) * d.C + (size_t)g0 * d.Cg;
}

// s: the sums of l, u, (l + u - 2 level)^2, (u - l)^2
__device__ __forceinline__ Box make_box(const Sum4& s, double level, const NormDims& d, double eps) {
    Box b;
    b.mean_l = s.a * d.inv_m;
    b.mean_u = s.b * d.inv_m;
    const double mc = (b.mean_l + b.mean_u) * 0.5 - level, vc = 0.25 * s.c * d.inv_m - mc * mc, vr = 0.25 * s.d * d.inv_m;
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

// A thread's sums into red: one for each channel, or one for its vector where that lies in one group.
template <int V>
__device__ __forceinline__ void put_sums(Sum4* red, const NormPlan& p, int rt, int cv, const Sum4 (&s)[V]) {
    if (p.same) {
        Sum4 t = s[0];
#pragma unroll
        for (int j = 1; j < V; ++j) t = add4(t, s[j]);
        red[rt * p.tx + cv] = t;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) red[(rt * p.tx + cv) * V + j] = s[j];
    }
}
// Adds the threads' sums of each group of the block up, one warp to a group; done(g, sum) in its lane 0.
template <typename Done>
__device__ __forceinline__ void group_sums(const Sum4* red, const NormDims& d, const NormPlan& p, const NormBlock& b, Done done) {
    const int per = (p.pieces == 1 ? d.Cg : b.nvec * p.V) / (p.same ? p.V : 1), width = p.same ? p.tx : p.tx * p.V;
    for (int g = threadIdx.x >> 5; g < b.ng; g += blockDim.x >> 5) {
        Sum4 t = {0.0, 0.0, 0.0, 0.0};
        for (int i = threadIdx.x & 31; i < per * p.rt; i += 32) {
            const int r = i / per;
            t = add4(t, red[r * width + g * per + (i - r * per)]);
        }
        t = warp_sum4(t);
        if ((threadIdx.x & 31) == 0) done(g, t);
    }
}
// What the elements of a group share in the backward pass.
struct Back {
    double s0, s1;              // means of the gradients at n- and n+
    double by_c, by_r;          // factor of c - mean(c), and of r
};
// from the group's sums of the gradients at n-, n+, s_lo, s_hi
__device__ __forceinline__ Back make_back(const Box& x, const Sum4& t, const NormDims& d) {
    Back k;
    k.s0 = t.a * d.inv_m;
    k.s1 = t.b * d.inv_m;
    const double lo = t.c * x.s_lo * x.s_lo * x.s_lo * (x.sd + x.rho), hi = t.d * x.s_hi * x.s_hi * x.s_hi * fmax(x.sd - x.rho, 0.0);
    // std and rho have no slope at 0, where all centres are one or all radii are 0: none is passed on
    k.by_c = x.sd > 0.0 ? -(lo + hi) * d.inv_m / x.sd : 0.0;
    k.by_r = x.rho > 0.0 ? (hi - lo) * d.inv_m / x.rho : 0.0;
    return k;
}

__device__ __forceinline__ int group_of(const NormDims& d, const NormPlan& p, int c) { return p.pieces == 1 ? p.by_cg(c) : 0; }

// Twice the levels of a column's channels (SAME: of its one group).
template <int V, bool SAME> struct Levels {
    double twice[SAME ? 1 : V];
    __device__ __forceinline__ Levels(const float* base, const NormDims& d, const NormPlan& p, int c) {
        if constexpr (SAME) {
            twice[0] = 2.0 * base[p.pieces == 1 ? p.by_cg(c) * d.Cg : 0];
        } else {
            int g[V];
            groups_of<V>(d, p, c, g);
#pragma unroll
            for (int j = 0; j < V; ++j) twice[j] = 2.0 * base[g[j] * d.Cg];
        }
    }
};

// Adds l, u, (l + u - 2 level)^2, (u - l)^2 of a vector up.
template <int V, bool SAME>
__device__ __forceinline__ void sum_vector(const Raw<float, V>& lv, const Raw<float, V>& uv, const Levels<V, SAME>& level, Sum4 (&s)[V]) {
    float l[V], u[V];
    unpack<float, V>(lv, l);
    unpack<float, V>(uv, u);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const double a = l[j], e = u[j];
        s[j].a += a;
        s[j].b += e;
        const double twice = a + e - level.twice[SAME ? 0 : j];
        s[j].c = ::fma(twice, twice, s[j].c);
        s[j].d = ::fma(e - a, e - a, s[j].d);
    }
}

// What the forward pass needs of a box, in fp32; the means as a sum of two.  far: differences from a mean may be beyond fp32, and s_lo and s_hi below its
// normal numbers: differences are taken as kFar of themselves then, s_lo and s_hi as 1 / kFar times theirs (both exact).
constexpr float kFar = 1.f / 16.f;
struct Ends32 { float ml, ml2, mu, mu2, s_lo, s_hi; bool far; };
__device__ __forceinline__ Ends32 make_ends32(const Sum4& s, double level, const NormDims& d, double eps) {
    const Box b = make_box(s, level, d, eps);
    Ends32 e;
    e.ml = (float)b.mean_l;
    e.ml2 = (float)(b.mean_l - e.ml);
    e.mu = (float)b.mean_u;
    e.mu2 = (float)(b.mean_u - e.mu);
    // |x - mean| <= sqrt(M) (sd + rho) at both ends, whose means are 2 rho apart at most: below 3 sqrt(M) (sd + rho), here 2e38 and more.  Not where
    // they are no number.  (A root here: 10.4 -> 12.4 us for bounds of 201 x 512.)
    const double most = b.sd + b.rho;
    e.far = most * most >= 5e75 * d.inv_m;
    e.s_lo = (float)(e.far ? b.s_lo / kFar : b.s_lo);
    e.s_hi = (float)(e.far ? b.s_hi / kFar : b.s_hi);
    return e;
}
// ... and of the channels of a thread's column; h: 1, or kFar where one of them has far ends
template <int V> struct BoundColumn { Ends32 e[V]; float w[V], o[V], inv_m2, cut, h; };
template <int V>
__device__ __forceinline__ void load_column(BoundColumn<V>& k, const Ends32* ends, const Param& gamma, const Param& beta, const NormDims& d,
                                            const NormPlan& p, const NormBlock& b, int c) {
    int g[V];
    groups_of<V>(d, p, c, g);
    load_params<V>(gamma, b.c0 + c, k.w);
    load_params<V>(beta, b.c0 + c, k.o);
#pragma unroll
    for (int j = 0; j < V; ++j) k.e[j] = ends[g[j]];
    bool far = false;
#pragma unroll
    for (int j = 0; j < V; ++j) far = far || k.e[j].far;
    k.h = far ? kFar : 1.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float up = far && !k.e[j].far ? 1.f / kFar : 1.f;
        k.e[j].s_lo *= up;
        k.e[j].s_hi *= up;
        k.e[j].ml *= k.h;
        k.e[j].ml2 *= k.h;
        k.e[j].mu *= k.h;
        k.e[j].mu2 *= k.h;
    }
    k.inv_m2 = 2.f * (float)d.inv_m * k.h;
    k.cut = sqrtf((float)((double)d.L * d.Cg - 1.0));
}

template <int V>
__device__ __forceinline__ void write_bounds(const Raw<float, V>& lv, const Raw<float, V>& uv, const BoundColumn<V>& k, size_t i, int act, float* out_l,
                                             float* out_u) {
    float l[V], u[V];
    unpack<float, V>(lv, l);
    unpack<float, V>(uv, u);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const Ends32& e = k.e[j];
        const float own = fmaf(u[j], 0.5f, -0.5f * l[j]) * k.inv_m2;      // the width halved: it may be beyond fp32
        const float n0 = (fmaf(l[j], k.h, -e.mu) - e.mu2) + own, n1 = (fmaf(u[j], k.h, -e.ml) - e.ml2) - own;
        float z0 = n0 * (n0 >= 0.f ? e.s_lo : e.s_hi), z1 = n1 * (n1 >= 0.f ? e.s_hi : e.s_lo);
        z0 = z0 <= -k.cut ? -k.cut : z0;                        // a NaN stays
        z1 = z1 >= k.cut ? k.cut : z1;
        const bool turned = k.w[j] < 0.f;
        const float v0 = fmaf(turned ? z1 : z0, k.w[j], k.o[j]), v1 = fmaf(turned ? z0 : z1, k.w[j], k.o[j]);
        float y0 = activate(v0, act), y1 = activate(v1, act);
        if (act == LINF_ACT_SILU) {
            const float low = v0 < kSiluArg && v1 > kSiluArg ? activate(kSiluArg, act) : y0, high = y0 > y1 ? y0 : y1;
            y0 = y1 < low ? y1 : low;
            y1 = high;
        }
        l[j] = y0;
        u[j] = y1;
    }
    store_once<float, V>(out_l + i, pack<float, V>(l));
    store_once<float, V>(out_u + i, pack<float, V>(u));
}

// Shared memory: the rows of `tensors` tensors, the threads' sums, then what the groups share.
struct BoundSpace { size_t red, box, back, bytes; };
template <int V>
__host__ __device__ inline BoundSpace bound_space(const NormPlan& p, int tensors) {
    BoundSpace s;
    const size_t four = sizeof(Sum4) * p.rt * p.tx * (p.same ? 1 : V), two = sizeof(double2) * p.rt * p.tx * V;
    s.red = tensors > 0 ? ((size_t)p.rows * p.tx * V * sizeof(float) * tensors + 15) / 16 * 16 : 0;
    s.box = s.red + ((four > two ? four : two) + 15) / 16 * 16;
    s.back = s.box + sizeof(Box) * p.groups;
    s.bytes = s.back + sizeof(Back) * p.groups;
    return s;
}

template <int V, bool SAME>
__global__ void __launch_bounds__(kNormThreads, 4)
bound_kept_kernel(const float* __restrict__ lower, const float* __restrict__ upper, Param gamma, Param beta, NormDims d, NormPlan p, double eps, int act,
                  float* __restrict__ out_l, float* __restrict__ out_u, Sum4* __restrict__ sums) {
    extern __shared__ uint4 space[];
    const BoundSpace at_ = bound_space<V>(p, 2);
    float* data = reinterpret_cast<float*>(space);
    Sum4* red = reinterpret_cast<Sum4*>(reinterpret_cast<char*>(space) + at_.red);
    Ends32* ends = reinterpret_cast<Ends32*>(reinterpret_cast<char*>(space) + at_.box);
    const int n = p.by_blocks(blockIdx.x);
    const NormBlock b = norm_block<V>(d, p, blockIdx.x - n * p.blocks);
    const int rt = p.by_tx(threadIdx.x), cv = threadIdx.x - rt * p.tx, c = cv * V;
    const bool in = rt < p.rt && cv < b.nvec;
    const int r1 = in ? d.L : 0, pitch = p.tx * V;
    const size_t at = ((size_t)n * d.L) * d.C + b.c0 + c;
    float* own_l = data + c;
    float* own_u = own_l + (size_t)p.rows * pitch;
    const Levels<V, SAME> level(level_of(lower, d, n, b.g0), d, p, in ? c : 0);
    for (int r = rt; r < r1; r += p.rt) {
        keep_vector<float, V>(own_l + r * pitch, lower + at + (size_t)r * d.C);
        keep_vector<float, V>(own_u + r * pitch, upper + at + (size_t)r * d.C);
    }
    keep_wait();
    if (in) {
        Sum4 s[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = Sum4{0.0, 0.0, 0.0, 0.0};
#pragma unroll 1
        for (int r = rt; r < r1; r += p.rt) sum_vector<V, SAME>(load_raw<float, V>(own_l + r * pitch), load_raw<float, V>(own_u + r * pitch), level, s);
        put_sums<V>(red, p, rt, cv, s);
    }
    __syncthreads();
    group_sums(red, d, p, b, [&](int g, const Sum4& s) {
        ends[g] = make_ends32(s, data[(d.L / 2) * pitch + g * d.Cg], d, eps);       // the level, as it was kept
        if (sums != nullptr) sums[(size_t)n * d.G + b.g0 + g] = s;
    });
    __syncthreads();
    if (in) {
        BoundColumn<V> col;
        load_column<V>(col, ends, gamma, beta, d, p, b, c);
#pragma unroll 2
        for (int r = rt; r < r1; r += p.rt)
            write_bounds<V>(load_raw<float, V>(own_l + r * pitch), load_raw<float, V>(own_u + r * pitch), col, at + (size_t)r * d.C, act, out_l, out_u);
    }
}

constexpr int kBoundRing = 4;              // rows that are on their way at a time

template <int V, bool SAME>
__global__ void __launch_bounds__(kNormThreads, 3)
bound_sums_kernel(const float* __restrict__ lower, const float* __restrict__ upper, NormDims d, NormPlan p, Sum4* __restrict__ part) {
    extern __shared__ uint4 space[];                            // the ring, then [rt][tx] or [rt][tx * V]
    Sum4* red4 = space_at<Sum4>(space, norm_ring_bytes<float, V, 2, kBoundRing>());
    const int n = p.by_blocks(blockIdx.x), split = blockIdx.y;
    const NormBlock b = norm_block<V>(d, p, blockIdx.x - n * p.blocks);
    const int rt = p.by_tx(threadIdx.x), cv = threadIdx.x - rt * p.tx;
    if (rt < p.rt && cv < b.nvec) {
        const size_t at = ((size_t)n * d.L) * d.C + b.c0 + cv * V;
        const float* const from[2] = {lower + at, upper + at};
        NormStream<float, V, 2, kBoundRing> stream(space, from, split * p.rt + rt, d.L, p.splits * p.rt, d.C);
        grid_let_go();
        const Levels<V, SAME> level(level_of(lower, d, n, b.g0), d, p, cv * V);
        Sum4 s[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = Sum4{0.0, 0.0, 0.0, 0.0};
        stream.template run<true>(rows_of(norm_rows(d, p, split), rt), [&](int, const Raw<float, V>(&v)[2]) { sum_vector<V, SAME>(v[0], v[1], level, s); });
        put_sums<V>(red4, p, rt, cv, s);
    }
    __syncthreads();
    group_sums(red4, d, p, b, [&](int g, const Sum4& s) { part[(((size_t)n * p.splits + split) * d.G + b.g0 + g) * p.pieces + b.piece] = s; });
}

// The sums of a group over the CTAs that share its rows and over its pieces, in all lanes.
__device__ __forceinline__ Sum4 all_parts(const Sum4* part, const NormDims& d, const NormPlan& p, int n, int g) {
    Sum4 t = {0.0, 0.0, 0.0, 0.0};
    for (int k = threadIdx.x & 31; k < p.splits * p.pieces; k += 32) {
        const int s = k / p.pieces, piece = k - s * p.pieces;
        const double2* v = reinterpret_cast<const double2*>(part + (((size_t)n * p.splits + s) * d.G + g) * p.pieces + piece);
        const double2 a = __ldcg(v), e = __ldcg(v + 1);
        t = add4(t, Sum4{a.x, a.y, e.x, e.y});
    }
    return warp_sum4(t);
}

template <int V>
__global__ void __launch_bounds__(kNormThreads, 3)
bound_apply_kernel(const float* __restrict__ lower, const float* __restrict__ upper, Param gamma, Param beta, const Sum4* __restrict__ part, NormDims d,
                   NormPlan p, double eps, int act, float* __restrict__ out_l, float* __restrict__ out_u, Sum4* __restrict__ sums) {
    extern __shared__ uint4 space[];                            // the ring, then what the groups share
    Ends32* ends = space_at<Ends32>(space, norm_ring_bytes<float, V, 2, kBoundRing>());
    const int last = gridDim.x - 1 - blockIdx.x, n = p.by_blocks(last), split = p.splits - 1 - blockIdx.y;
    const NormBlock b = norm_block<V>(d, p, last - n * p.blocks);
    const int rt = p.by_tx(threadIdx.x), cv = threadIdx.x - rt * p.tx;
    const bool in = rt < p.rt && cv < b.nvec;
    const size_t at = ((size_t)n * d.L) * d.C + b.c0 + cv * V;
    const float* const from[2] = {lower + at, upper + at};
    NormStream<float, V, 2, kBoundRing> stream(space, from, split * p.rt + rt, in ? d.L : 0, p.splits * p.rt, d.C);
    const float* base = level_of(lower, d, n, b.g0);
    grid_wait();
    for (int g = threadIdx.x >> 5; g < b.ng; g += kNormThreads / 32) {
        const float level = base[(size_t)g * d.Cg];
        const Sum4 t = all_parts(part, d, p, n, b.g0 + g);
        if ((threadIdx.x & 31) == 0) {
            ends[g] = make_ends32(t, level, d, eps);
            if (split == 0 && b.piece == 0 && sums != nullptr) sums[(size_t)n * d.G + b.g0 + g] = t;
        }
    }
    __syncthreads();
    if (!in) return;
    BoundColumn<V> col;
    load_column<V>(col, ends, gamma, beta, d, p, b, cv * V);
    stream.run_all([&](int r, const Raw<float, V>(&v)[2]) {
        write_bounds<V>(v[0], v[1], col, at + (size_t)r * d.C, act, out_l, out_u);
    });
}

// ---- backward -----------------------------------------------------------------------------------------------------

// gradients at z- and z+ of one element, and what they add to those of gamma and beta
__device__ __forceinline__ void bound_dz(const Ends& e, float w, float o, int act, float g0, float g1, double& q0, double& q1, double& dw, double& db) {
    const bool turned = w < 0.f;
    const double z0 = turned ? e.z1 : e.z0, z1 = turned ? e.z0 : e.z1;
    double d0, d1;
    bound_slope(::fma(z0, (double)w, (double)o), ::fma(z1, (double)w, (double)o), act, g0, g1, d0, d1);
    dw = d0 * z0 + d1 * z1;
    db = d0 + d1;
    q0 = e.cut0 ? 0.0 : (turned ? d1 : d0) * (double)w;
    q1 = e.cut1 ? 0.0 : (turned ? d0 : d1) * (double)w;
}


struct In4 { const float *g_l, *g_u, *lower, *upper; };

// What one vector adds to its group's sums (gradients at n-, n+, s_lo, s_hi) and to its channels' (beta, gamma).
template <int V>
__device__ __forceinline__ void sum_back(const Raw<float, V>& lv, const Raw<float, V>& uv, const Raw<float, V>& glv, const Raw<float, V>& guv,
                                         const Box* box, const float (&w)[V], const float (&o)[V], const NormDims& d, const NormPlan& p, int c, int act,
                                         Sum4 (&s)[V], double2 (&by)[V]) {
    float l[V], u[V], gl[V], gu[V];
    unpack<float, V>(lv, l);
    unpack<float, V>(uv, u);
    unpack<float, V>(glv, gl);
    unpack<float, V>(guv, gu);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const Ends e = make_ends(box[group_of(d, p, c + j)], l[j], u[j], d.inv_m);
        double q0, q1, dw, db;
        bound_dz(e, w[j], o[j], act, gl[j], gu[j], q0, q1, dw, db);
        by[j].x += db;
        by[j].y += dw;
        s[j].a = ::fma(q0, e.s0, s[j].a);
        s[j].b = ::fma(q1, e.s1, s[j].b);
        const double t0 = q0 * e.n0, t1 = q1 * e.n1;
        s[j].c += (e.n0 >= 0.0 ? t0 : 0.0) + (e.n1 >= 0.0 ? 0.0 : t1);
        s[j].d += (e.n0 >= 0.0 ? 0.0 : t0) + (e.n1 >= 0.0 ? t1 : 0.0);
    }
}

template <int V>
__device__ __forceinline__ void write_back(const Raw<float, V>& lv, const Raw<float, V>& uv, const Raw<float, V>& glv, const Raw<float, V>& guv,
                                           const Box* box, const Back* back, const float (&w)[V], const float (&o)[V], const NormDims& d,
                                           const NormPlan& p, int c, size_t i, int act, float* d_l, float* d_u) {
    float l[V], u[V], gl[V], gu[V];
    unpack<float, V>(lv, l);
    unpack<float, V>(uv, u);
    unpack<float, V>(glv, gl);
    unpack<float, V>(guv, gu);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int g = group_of(d, p, c + j);
        const Box& x = box[g];
        const Back& m = back[g];
        const double a = l[j], e = u[j];
        const Ends s = make_ends(x, a, e, d.inv_m);
        double q0, q1, dw, db;
        bound_dz(s, w[j], o[j], act, gl[j], gu[j], q0, q1, dw, db);
        q0 *= s.s0;
        q1 *= s.s1;
        const double dc = m.by_c * ((a + e) - (x.mean_l + x.mean_u)) * 0.5, dr = m.by_r * (e - a) * 0.5;
        gl[j] = (float)(q0 + (q1 - q0) * d.inv_m - m.s1 + (dc - dr) * 0.5);
        gu[j] = (float)(q1 + (q0 - q1) * d.inv_m - m.s0 + (dc + dr) * 0.5);
    }
    store_once<float, V>(d_l + i, pack<float, V>(gl));
    store_once<float, V>(d_u + i, pack<float, V>(gu));
}

// Per-channel sums of a CTA's threads, added up along the rows and written to `to`; red is free before and after.
template <int V>
__device__ __forceinline__ void put_channels(double2* red, const NormPlan& p, const NormBlock& b, int rt, int cv, const double2 (&by)[V], float2* to) {
    const int width = p.tx * V;
    __syncthreads();
    if (rt < p.rt) {
#pragma unroll
        for (int j = 0; j < V; ++j) red[rt * width + cv * V + j] = by[j];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < b.nvec * V; c += blockDim.x) {
        double s = 0.0, t = 0.0;
        for (int r = 0; r < p.rt; ++r) { s += red[r * width + c].x; t += red[r * width + c].y; }
        __stcg(to + c, make_float2((float)s, (float)t));
    }
    __syncthreads();
}

template <int V>
__global__ void __launch_bounds__(kNormThreads, 2)
bound_back_kept_kernel(In4 in4, Param gamma, Param beta, const Sum4* __restrict__ sums, NormDims d, NormPlan p, double eps, int act,
                       float* __restrict__ d_l, float* __restrict__ d_u, float2* __restrict__ by_channel) {
    extern __shared__ uint4 space[];
    const BoundSpace at_ = bound_space<V>(p, 4);
    float* data = reinterpret_cast<float*>(space);
    Sum4* red = reinterpret_cast<Sum4*>(reinterpret_cast<char*>(space) + at_.red);
    Box* box = reinterpret_cast<Box*>(reinterpret_cast<char*>(space) + at_.box);
    Back* back = reinterpret_cast<Back*>(reinterpret_cast<char*>(space) + at_.back);
    const int chunk = p.by_blocks(blockIdx.x);
    const NormBlock b = norm_block<V>(d, p, blockIdx.x - chunk * p.blocks);
    const int rt = p.by_tx(threadIdx.x), cv = threadIdx.x - rt * p.tx, c = cv * V;
    const bool in = rt < p.rt && cv < b.nvec;
    const int r1 = in ? d.L : 0, pitch = p.tx * V;
    const int n1 = min(d.N, (chunk + 1) * p.per_cta);
    const size_t tensor = (size_t)p.rows * pitch;
    float* own = data + c;                                      // lower, upper and their gradients, one behind the other
    float w[V], o[V];
    double2 by[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        w[j] = in ? load_param(gamma, b.c0 + c + j) : 1.f;
        o[j] = in ? load_param(beta, b.c0 + c + j) : 0.f;
        by[j] = make_double2(0.0, 0.0);
    }
    for (int n = chunk * p.per_cta; n < n1; ++n) {
        const size_t at = ((size_t)n * d.L) * d.C + b.c0 + c;
        for (int r = rt; r < r1; r += p.rt) {
            const size_t i = at + (size_t)r * d.C;
            keep_vector<float, V>(own + r * pitch, in4.lower + i);
            keep_vector<float, V>(own + tensor + r * pitch, in4.upper + i);
            keep_vector<float, V>(own + 2 * tensor + r * pitch, in4.g_l + i);
            keep_vector<float, V>(own + 3 * tensor + r * pitch, in4.g_u + i);
        }
        for (int g = threadIdx.x; g < b.ng; g += blockDim.x) box[g] = make_box(sums[(size_t)n * d.G + b.g0 + g], level_of(in4.lower, d, n, b.g0)[(size_t)g * d.Cg], d, eps);
        keep_wait();
        __syncthreads();
        if (in) {
            Sum4 s[V];
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] = Sum4{0.0, 0.0, 0.0, 0.0};
            for (int r = rt; r < r1; r += p.rt) {
                const float* at_r = own + r * pitch;
                sum_back<V>(load_raw<float, V>(at_r), load_raw<float, V>(at_r + tensor), load_raw<float, V>(at_r + 2 * tensor),
                            load_raw<float, V>(at_r + 3 * tensor), box, w, o, d, p, c, act, s, by);
            }
            put_sums<V>(red, p, rt, cv, s);
        }
        __syncthreads();
        if (d_l == nullptr) continue;                           // the same for every thread
        group_sums(red, d, p, b, [&](int g, const Sum4& s) { back[g] = make_back(box[g], s, d); });
        __syncthreads();
        if (in)
            for (int r = rt; r < r1; r += p.rt) {
                const float* at_r = own + r * pitch;
                write_back<V>(load_raw<float, V>(at_r), load_raw<float, V>(at_r + tensor), load_raw<float, V>(at_r + 2 * tensor),
                              load_raw<float, V>(at_r + 3 * tensor), box, back, w, o, d, p, c, at + (size_t)r * d.C, act, d_l, d_u);
            }
        __syncthreads();
    }
    put_channels<V>(reinterpret_cast<double2*>(red), p, b, rt, cv, by, by_channel + (size_t)chunk * d.C + b.c0);
}

template <int V>
__global__ void __launch_bounds__(kNormThreads, 2)
bound_back_sums_kernel(In4 in4, Param gamma, Param beta, const Sum4* __restrict__ sums, NormDims d, NormPlan p, double eps, int act,
                       float2* __restrict__ by_channel, Sum4* __restrict__ by_group) {
    extern __shared__ uint4 space[];
    const BoundSpace at_ = bound_space<V>(p, 0);
    Sum4* red = reinterpret_cast<Sum4*>(space);
    Box* box = reinterpret_cast<Box*>(reinterpret_cast<char*>(space) + at_.box);
    const int n = p.by_blocks(blockIdx.x), split = blockIdx.y;
    const NormBlock b = norm_block<V>(d, p, blockIdx.x - n * p.blocks);
    for (int g = threadIdx.x; g < b.ng; g += kNormThreads) box[g] = make_box(sums[(size_t)n * d.G + b.g0 + g], level_of(in4.lower, d, n, b.g0)[(size_t)g * d.Cg], d, eps);
    __syncthreads();
    const int rt = p.by_tx(threadIdx.x), cv = threadIdx.x - rt * p.tx, c = cv * V;
    const bool in = rt < p.rt && cv < b.nvec;
    Sum4 s[V];
    double2 by[V];
#pragma unroll
    for (int j = 0; j < V; ++j) { s[j] = Sum4{0.0, 0.0, 0.0, 0.0}; by[j] = make_double2(0.0, 0.0); }
    if (in) {
        float w[V], o[V];
        load_params<V>(gamma, b.c0 + c, w);
        load_params<V>(beta, b.c0 + c, o);
        const size_t at = ((size_t)n * d.L) * d.C + b.c0 + c;
        for (int r = split * p.rt + rt; r < d.L; r += p.splits * p.rt) {
            const size_t i = at + (size_t)r * d.C;
            sum_back<V>(load_raw<float, V>(in4.lower + i), load_raw<float, V>(in4.upper + i), load_raw<float, V>(in4.g_l + i),
                        load_raw<float, V>(in4.g_u + i), box, w, o, d, p, c, act, s, by);
        }
    }
    put_channels<V>(reinterpret_cast<double2*>(red), p, b, rt, cv, by, by_channel + ((size_t)n * p.splits + split) * d.C + b.c0);
    if (in) put_sums<V>(red, p, rt, cv, s);
    __syncthreads();
    group_sums(red, d, p, b, [&](int g, const Sum4& q) { by_group[(((size_t)n * p.splits + split) * d.G + b.g0 + g) * p.pieces + b.piece] = q; });
}

template <int V>
__global__ void __launch_bounds__(kNormThreads)
bound_back_apply_kernel(In4 in4, Param gamma, Param beta, const Sum4* __restrict__ sums, const Sum4* __restrict__ by_group, NormDims d, NormPlan p,
                        double eps, int act, float* __restrict__ d_l, float* __restrict__ d_u) {
    extern __shared__ uint4 space[];
    const BoundSpace at_ = bound_space<V>(p, 0);
    Box* box = reinterpret_cast<Box*>(reinterpret_cast<char*>(space) + at_.box);
    Back* back = reinterpret_cast<Back*>(reinterpret_cast<char*>(space) + at_.back);
    const int last = gridDim.x - 1 - blockIdx.x, n = p.by_blocks(last), split = p.splits - 1 - blockIdx.y;
    const NormBlock b = norm_block<V>(d, p, last - n * p.blocks);
    grid_wait();
    for (int g = threadIdx.x >> 5; g < b.ng; g += kNormThreads / 32) {
        const Sum4 t = all_parts(by_group, d, p, n, b.g0 + g);
        if ((threadIdx.x & 31) == 0) {
            const Box x = make_box(sums[(size_t)n * d.G + b.g0 + g], level_of(in4.lower, d, n, b.g0)[(size_t)g * d.Cg], d, eps);
            box[g] = x;
            back[g] = make_back(x, t, d);
        }
    }
    __syncthreads();
    const int rt = p.by_tx(threadIdx.x), cv = threadIdx.x - rt * p.tx, c = cv * V;
    if (rt >= p.rt || cv >= b.nvec) return;
    float w[V], o[V];
    load_params<V>(gamma, b.c0 + c, w);
    load_params<V>(beta, b.c0 + c, o);
    const size_t at = ((size_t)n * d.L) * d.C + b.c0 + c;
    for (int r = split * p.rt + rt; r < d.L; r += p.splits * p.rt) {
        const size_t i = at + (size_t)r * d.C;
        write_back<V>(load_raw<float, V>(in4.lower + i), load_raw<float, V>(in4.upper + i), load_raw<float, V>(in4.g_l + i),
                      load_raw<float, V>(in4.g_u + i), box, back, w, o, d, p, c, i, act, d_l, d_u);
    }
}

// ---- launches -----------------------------------------------------------------------------------------------------

NormKind bound_kind(bool back) { return {4, back ? 4 : 2, back}; }

size_t parts_bytes(const NormDims& d, const NormPlan& p) { return p.kept ? 0 : sizeof(Sum4) * (size_t)d.N * p.splits * d.G * p.pieces; }
long long channel_rows(const NormPlan& p) { return (long long)p.chunks * p.splits; }
size_t workspace(const NormDims& d, const NormPlan& p, bool back) {
    return parts_bytes(d, p) + (back ? sizeof(float2) * (size_t)channel_rows(p) * d.C : 0);
}

template <int V, bool SAME>
int forward_as(const float* lower, const float* upper, const NormGiven& given, const NormDims& d, const NormPlan& p, double eps, int act, float* out_l,
               float* out_u, Sum4* sums, void* ws, cudaStream_t st) {
    if (p.kept)
        return launch_kept<bound_kept_kernel<V, SAME>>(p, bound_space<V>(p, 2).bytes, st, lower, upper, given.gamma, given.beta, d, p, eps, act, out_l,
                           out_u, sums);
    const dim3 grid((unsigned)(p.blocks * d.N), p.splits);
    Sum4* part = static_cast<Sum4*>(ws);
    const size_t ring = norm_ring_bytes<float, V, 2, kBoundRing>(), one = ring + bound_space<V>(p, 0).box, two = ring + sizeof(Ends32) * p.groups;
    if (!allow_shared<bound_sums_kernel<V, SAME>>(one) || !allow_shared<bound_apply_kernel<V>>(two)) return LINF_ERR_LAUNCH;
    bound_sums_kernel<V, SAME><<<grid, kNormThreads, one, st>>>(lower, upper, d, p, part);
    if (launch_status()) return LINF_ERR_LAUNCH;
    return launch_behind(bound_apply_kernel<V>, grid, kNormThreads, two, st, lower, upper, given.gamma, given.beta, part, d, p, eps, act, out_l, out_u,
                         sums);
}
template <int V>
int forward(const float* lower, const float* upper, const NormGiven& given, const NormDims& d, const NormPlan& p, double eps, int act, float* out_l,
            float* out_u, Sum4* sums, void* ws, cudaStream_t st) {
    if constexpr (V > 1)
        if (!p.same) return forward_as<V, false>(lower, upper, given, d, p, eps, act, out_l, out_u, sums, ws, st);
    return forward_as<V, true>(lower, upper, given, d, p, eps, act, out_l, out_u, sums, ws, st);
}

template <int V>
int backward(const In4& in4, const NormGiven& given, const Sum4* sums, const NormDims& d, const NormPlan& p, double eps, int act, float* d_l,
             float* d_u, float* dgamma, float* dbeta, void* ws, cudaStream_t st) {
    Sum4* by_group = static_cast<Sum4*>(ws);
    float2* by_channel = reinterpret_cast<float2*>(static_cast<char*>(ws) + parts_bytes(d, p));
    if (p.kept) {
        const int rc = launch_kept<bound_back_kept_kernel<V>>(p, bound_space<V>(p, 4).bytes, st, in4, given.gamma, given.beta, sums, d, p, eps,
                                   act, d_l, d_u, by_channel);
        if (rc) return rc;
    } else {
        const dim3 grid((unsigned)(p.blocks * d.N), p.splits);
        const size_t shared = bound_space<V>(p, 0).bytes;
        if (!allow_shared<bound_back_sums_kernel<V>>(shared) || !allow_shared<bound_back_apply_kernel<V>>(shared)) return LINF_ERR_LAUNCH;
        bound_back_sums_kernel<V><<<grid, kNormThreads, shared, st>>>(in4, given.gamma, given.beta, sums, d, p, eps, act, by_channel, by_group);
        if (launch_status()) return LINF_ERR_LAUNCH;
        if (d_l != nullptr) {
            const int rc = launch_behind(bound_back_apply_kernel<V>, grid, kNormThreads, shared, st, in4, given.gamma, given.beta, sums, by_group, d, p, eps,
                                         act, d_l, d_u);
            if (rc) return rc;
        }
    }
    return dgamma != nullptr || dbeta != nullptr ? norm_params(by_channel, channel_rows(p), d.C, dgamma, dbeta, LINF_F32, st) : LINF_OK;
}

}  // namespace

size_t group_norm_bound_workspace(int N, int C, int G, int L, bool back) {
    size_t most = 0;
    for (int k = 0; k < 2; ++k) {
        NormDims d;
        NormPlan p;
        if (norm_make(N, C, G, L, bound_kind(back), k == 0, &d, &p) != LINF_OK) return 0;
        const size_t need = workspace(d, p, back);
        if (need > most) most = need;
    }
    return (most + 255) / 256 * 256;
}

int group_norm_bound_forward(const float* lower, const float* upper, const float* gamma, const float* beta, int N, int C, int G, int L, double eps,
                             int act, float* out_l, float* out_u, double* sums, void* ws, size_t ws_bytes, cudaStream_t st) {
    NormDims d;
    NormPlan p;
    const int rc = norm_make(N, C, G, L, bound_kind(false), aligned16(lower) && aligned16(upper) && aligned16(out_l) && aligned16(out_u), &d, &p);
    if (rc) return rc;
    const size_t need = workspace(d, p, false);
    if (need > 0 && (ws == nullptr || !aligned16(ws) || ws_bytes < need)) return LINF_ERR_WORKSPACE;
    NormGiven given;
    if (!norm_given(gamma, beta, LINF_F32, &given)) return LINF_ERR_LAUNCH;
    Sum4* s = reinterpret_cast<Sum4*>(sums);
    return p.V == 4 ? forward<4>(lower, upper, given, d, p, eps, act, out_l, out_u, s, ws, st)
           : p.V == 2 ? forward<2>(lower, upper, given, d, p, eps, act, out_l, out_u, s, ws, st)
                      : forward<1>(lower, upper, given, d, p, eps, act, out_l, out_u, s, ws, st);
}

int group_norm_bound_backward(const float* g_l, const float* g_u, const float* lower, const float* upper, const float* gamma, const float* beta,
                              const double* sums, int N, int C, int G, int L, double eps, int act, float* d_l, float* d_u, float* dgamma,
                              float* dbeta, void* ws, size_t ws_bytes, cudaStream_t st) {
    NormDims d;
    NormPlan p;
    const int rc = norm_make(N, C, G, L, bound_kind(true),
                             aligned16(g_l) && aligned16(g_u) && aligned16(lower) && aligned16(upper) && aligned16(d_l) && aligned16(d_u), &d, &p);
    if (rc) return rc;
    const size_t need = workspace(d, p, true);
    if (ws == nullptr || !aligned16(ws) || ws_bytes < need) return LINF_ERR_WORKSPACE;
    NormGiven given;
    if (!norm_given(gamma, beta, LINF_F32, &given)) return LINF_ERR_LAUNCH;
    const Sum4* s = reinterpret_cast<const Sum4*>(sums);
    const In4 in4 = {g_l, g_u, lower, upper};
    return p.V == 4 ? backward<4>(in4, given, s, d, p, eps, act, d_l, d_u, dgamma, dbeta, ws, st)
           : p.V == 2 ? backward<2>(in4, given, s, d, p, eps, act, d_l, d_u, dgamma, dbeta, ws, st)
                      : backward<1>(in4, given, s, d, p, eps, act, d_l, d_u, dgamma, dbeta, ws, st);
}

}  // namespace linf
