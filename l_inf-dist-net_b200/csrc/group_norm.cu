// Group norm over channels-last activations x [N, L, C], with the activation and the dropout behind it in the same pass:
//   h = (x - mean) / sqrt(var + eps) over the L * C/G values of a sample's group,  u = gamma h + beta,  y = dropout(f(u))
// and its gradients: with du = dropout(dy) f'(u),
//   dbeta = sum du, dgamma = sum du h (over samples and positions),
//   dx = (gamma du - mean(gamma du) - h mean(gamma du h)) / sqrt(var + eps)
//
// What bounds it: kept and dense slabs the latency of load, reduction and store; two passes latency as well, at 14 to 28 warps on an SM: a bf16
// value with silu takes 12 to 15 instructions, with dropout 25, and 1.1 to 2.1 of 4 a clock are issued, while HBM, which sees x once or
// twice, is at 31 to 51 % of its peak.  Measured on one B200, us: 32 x 320 x 64 x 64 bf16, 32 groups, silu: 57 (sums 21, results 40 one by one and
// from HBM; 26 if x and y crossed HBM once); 16 x 128 x 160 x 160 bf16, silu and dropout: forward 83, backward 134; 64 x 128 x 16 x 16 fp32,
// tanh, kept: forward 10, backward 19.  Clusters of up to 8 CTAs that held larger slabs in
// their shared memory read x once, but loaded, reduced and stored in turn: 65 for the first, and 528 instead of 216 for the second, whose rows
// they had to cut into pieces of 32 bytes.
//
// The forward sums are fp32 over a few dozen rows of a thread, about a shift near the data, joined as means and variances, and 64-bit over the
// CTAs of a group (Moments).  So neither the number of rows, nor data far from 0 against their spread (activations of distance layers are all
// positive), nor single rows far from the others cost more than a few roundings.  The order of every addition is fixed by the shape alone.
#include "group_norm.cuh"

namespace linf {
namespace {

// The values that stand for a gamma or beta that was not given, and for the state of a generator that nothing is drawn from.
struct Own { float one, zero; long long rng[2]; };
__device__ Own g_own = {1.f, 0.f, {0, 0}};

// Mean (in two parts: values far from 0 against their spread would see the rounding of one) and 1 / deviation of a group.
struct alignas(16) Stat { float mean, rest, r; };
// What a thread's column needs for u = (x + m) a + o: m is the mean's first part with its sign turned, o takes the second.
template <int V> struct Column { Lanes<V> m, a, o; };
template <int V>
__device__ __forceinline__ void load_column(Column<V>& k, const Stat* stat, const Param& gamma, const Param& beta, const NormDims& d,
                                            const NormPlan& p, const NormBlock& b, int cv) {
    int g[V];
    groups_of<V>(d, p, cv * V, g);
    float m[V], a[V], o[V];
    load_params<V>(gamma, b.c0 + cv * V, a);
    load_params<V>(beta, b.c0 + cv * V, o);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const Stat s = stat[g[j]];
        m[j] = -s.mean;
        a[j] *= s.r;
        o[j] = fmaf(-s.rest, a[j], o[j]);
    }
    k.m.set(m);
    k.a.set(a);
    k.o.set(o);
}
template <typename T, int V>
__device__ __forceinline__ void write_vector(const Raw<T, V>& v, const Column<V>& col, int act, const Drop& drop, const DropKey& key, size_t i, T* y) {
    Lanes<V> u = activate<sizeof(T) == 4, V>(fma(add(lanes_of<T, V>(v), col.m), col.a, col.o), act);
    if (drop.on) u = linf::drop<V>(drop, key, i, u);
    store_once<T, V>(y + i, raw_of<T, V>(u));
}
__device__ __forceinline__ Stat finish_stat(double mean, double var, double eps) {
    Stat s;
    s.mean = (float)mean;
    s.rest = (float)(mean - (double)s.mean);
    s.r = 1.f / sqrtf((float)((var > 0.0 || var != var ? var : 0.0) + eps));
    return s;
}

// A thread's sums for the mean and the variance of what it reads.  They are taken in runs of at most 32 rows (8 the first time) about a shift near
// the data -- the first row, then the mean so far --, and the runs are added up: so a column's length costs few roundings, and a first row
// apart from the rest (a border, a special position) is as good as forgotten from the second run on.  A new shift: sums S, Q of n values,
// moved by e, become S + n e and Q + e (2 S + n e).  What a thread hands on is a shift, the mean less that shift, and the variance: data far
// from 0 against their spread lose nothing by the mean's rounding.
//   SAME (a vector lies in one group): one shift and one pair of sums for the vector; else one for each channel, the runs' in shared memory.
constexpr int kFirstRun = 8, kRun = 32;    // multiples of kRing
struct Part { float shift, mean, var; };   // of some values; the mean is shift + mean
template <int V, bool SAME> struct Moments {
    static_assert(SAME || V > 1, "a vector of one channel lies in one group");
    Lanes<V> k, s, q;                           // the shift with its sign turned, sum (x + k), sum (x + k)^2 of the run
    float S, Q;                                 // SAME: of the runs before
    float2* runs;                               // else: S, Q of each channel
    int rows;                                   // up to the last flush
    // place: where the thread's parts will be; its runs are there before
    __device__ __forceinline__ explicit Moments(Part* place) : S(0.f), Q(0.f), runs(reinterpret_cast<float2*>(place)), rows(0) {
        k = s = q = filled<V>(0.f);
    }
    __device__ __forceinline__ void start(const Lanes<V>& v) {
        if constexpr (SAME) {
            float f[V];
            mul(v, filled<V>(-1.f / V)).get(f);
            k = filled<V>(tree(f));
        } else {
            k = mul(v, filled<V>(-1.f));
        }
    }
    __device__ __forceinline__ void add(const Lanes<V>& v) {
        const Lanes<V> e = linf::add(v, k);
        s = linf::add(s, e);
        q = fma(e, e, q);
    }
    // what came since the last flush; upto: rows so far
    __device__ __forceinline__ void flush(int upto) {
        if constexpr (SAME) {
            float a, b;
            all_runs(a, b);
            rows = upto;
            const float n = (float)(rows * V), from = shift(), to = fmaf(a, -1.f / n, from), e = to - from;
            S = fmaf(n, e, a);
            Q = fmaf(e, a + S, b);
            k = filled<V>(to);
        } else {
            Lanes<V> a, b;
            all_runs(a, b);
            rows = upto;
            const Lanes<V> to = fma(a, filled<V>(-1.f / (float)rows), k), e = fma(k, filled<V>(-1.f), to);
            const Lanes<V> moved = fma(e, filled<V>((float)rows), a);
            float f[V], h[V];
            moved.get(f);
            fma(e, linf::add(a, moved), b).get(h);
#pragma unroll
            for (int j = 0; j < V; ++j) runs[j] = make_float2(f[j], h[j]);
            k = to;
        }
        s = q = filled<V>(0.f);
    }
    // mean and variance of `all` rows, for each channel or for the vector
    __device__ __forceinline__ void put(Part* to, int all) const {
        if constexpr (SAME) {
            float a, b;
            all_runs(a, b);
            const float inv = 1.f / (float)(all * V), m = a * inv;
            *to = Part{-shift(), m, fmaf(-m, m, b * inv)};
        } else {
            Lanes<V> a, b;
            all_runs(a, b);
            const Lanes<V> inv = filled<V>(1.f / (float)all);
            float m[V], v[V], h[V];
            mul(a, inv).get(m);
            mul(b, inv).get(v);
            k.get(h);
#pragma unroll
            for (int j = 0; j < V; ++j) to[j] = Part{-h[j], m[j], fmaf(-m[j], m[j], v[j])};
        }
    }
private:
    static __device__ __forceinline__ float tree(float (&f)[V]) {
#pragma unroll
        for (int n = V / 2; n > 0; n /= 2)
#pragma unroll
            for (int j = 0; j < n; ++j) f[j] += f[j + n];
        return f[0];
    }
    __device__ __forceinline__ float shift() const { float f[V]; k.get(f); return f[0]; }
    // the sums of all rows so far about the shift
    __device__ __forceinline__ void all_runs(float& a, float& b) const {
        float f[V], h[V];
        s.get(f);
        q.get(h);
        a = S + tree(f);
        b = Q + tree(h);
    }
    __device__ __forceinline__ void all_runs(Lanes<V>& a, Lanes<V>& b) const {
        a = s;
        b = q;
        if (rows == 0) return;
        float f[V], h[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float2 v = runs[j];
            f[j] = v.x;
            h[j] = v.y;
        }
        a = linf::add(lanes<V>(f), s);
        b = linf::add(lanes<V>(h), q);
    }
};
// A thread's place among the CTA's parts.
template <int V, bool SAME> __device__ __forceinline__ Part* moments_at(Part* red, const NormPlan& p, int rt, int cv) {
    return red + (rt * p.tx + cv) * (SAME ? 1 : V);
}

// Mean and variance of each group of the block over the CTA's rows from what the threads put into red; done(g, mean, variance) in one lane.
// Parts of weights w_i join as mean = sum w_i mean_i, variance = sum w_i (variance_i + mean_i^2) - mean^2, about one part's mean.
template <int V, bool SAME, typename Done>
__device__ __forceinline__ void join_moments(Part* red, const NormDims& d, const NormPlan& p, const NormBlock& b, const NormRows& share, Done done) {
    const int width = SAME ? p.tx : p.tx * V, lane = threadIdx.x & 31;
    const int per = (p.pieces == 1 ? d.Cg : b.nvec * V) / (SAME ? V : 1);         // columns of red of a group
    __syncthreads();
    if (p.rt > 1) {
        // columns along the rows
        by_columns(width, p.rt, [&](int c, int first, int step, auto join) {
            const float k0 = c < width ? red[c].shift + red[c].mean : 0.f, inv = 1.f / (float)share.all;
            float s = 0.f, q = 0.f;
            for (int r = first; r < p.rt; r += step) {
                const Part v = red[r * width + c];
                const float weight = (float)rows_of(share, r) * inv, e = (v.shift - k0) + v.mean;
                s = fmaf(weight, e, s);
                q = fmaf(weight, fmaf(e, e, v.var), q);
            }
            if (join(s, q)) red[c] = Part{k0, s, fmaf(-s, s, q)};
        });
        __syncthreads();
    }
    // groups along their columns: as many lanes to a group as the group has columns, up to a warp
    int wide = 1;
    while (wide < per && wide < 32) wide *= 2;
    const float by = 1.f / (float)per;
    for (int g0 = (threadIdx.x >> 5) * (32 / wide); g0 < b.ng; g0 += (blockDim.x >> 5) * (32 / wide)) {
        const int g = g0 + lane / wide;
        float s = 0.f, q = 0.f, k0 = 0.f;
        if (g < b.ng) {
            k0 = red[g * per].shift + red[g * per].mean;
            for (int c = lane & (wide - 1); c < per; c += wide) {
                const Part v = red[g * per + c];
                const float e = (v.shift - k0) + v.mean;
                s += e;
                q += fmaf(e, e, v.var);
            }
        }
        for (int o = 1; o < wide; o *= 2) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            q += __shfl_xor_sync(0xffffffffu, q, o);
        }
        s *= by;
        if (g < b.ng && (lane & (wide - 1)) == 0) done(g, (double)k0 + (double)s, fmaf(-s, s, q * by));
    }
}

// ---- forward, kept --------------------------------------------------------------------------------------------------

// Shared memory: the rows of all tensors, a pair for each thread and channel (or vector), the statistics of each group, and where elements are
// dropped in a backward pass a byte for each vector: which of its elements are kept.  Offsets in bytes.
struct KeptSpace { int red, stat, mask, bytes; };
KeptSpace kept_space(const NormPlan& p, int elem_bytes, int tensors, size_t of_thread, bool by_vector, size_t of_group, bool masks) {
    KeptSpace s;
    s.red = (p.rows * p.tx * p.V * elem_bytes * tensors + 15) / 16 * 16;
    s.stat = (s.red + (int)of_thread * p.rt * p.tx * (by_vector ? 1 : p.V) + 15) / 16 * 16;
    s.mask = s.stat + (int)of_group * p.groups;
    s.bytes = s.mask + (masks ? p.rows * p.tx : 0);
    return s;
}

template <typename T, int V, bool SAME>
__global__ void __launch_bounds__(kNormThreads, 3)
norm_kept_kernel(const T* __restrict__ x, Param gamma, Param beta, NormDims d, NormPlan p, KeptSpace sp, double eps, int act, Drop drop,
                 T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
    extern __shared__ uint4 space[];
    T* data = reinterpret_cast<T*>(space);
    Part* red = space_at<Part>(space, sp.red);
    Stat* stat = space_at<Stat>(space, sp.stat);
    const int n = p.by_blocks(blockIdx.x);
    const NormBlock b = norm_block<V>(d, p, blockIdx.x - n * p.blocks);
    const int rt = p.by_tx(threadIdx.x), cv = threadIdx.x - rt * p.tx;
    const bool in = rt < p.rt && cv < b.nvec;
    const int r1 = in ? d.L : 0;
    const NormRows share = norm_rows(d, p, 0);
    const size_t at = ((size_t)n * d.L) * d.C + b.c0 + cv * V;
    T* own = data + cv * V;
    const int pitch = p.tx * V;
    for (int r = rt; r < r1; r += p.rt) keep_vector<T, V>(own + r * pitch, x + at + (size_t)r * d.C);
    keep_wait();
    if (in) {
        Part* place = moments_at<V, SAME>(red, p, rt, cv);
        Moments<V, SAME> t(place);
        t.start(load_lanes<T, V>(own + rt * pitch));
        const int rows = rows_of(share, rt);
        const T* at_r = own + rt * pitch;
        for (int r = 0, run = kFirstRun; r < rows; run = kRun) {
            const int to = min(rows, r + run);
#pragma unroll 4
            for (; r < to; ++r, at_r += p.rt * pitch) t.add(load_lanes<T, V>(at_r));
            if (to < rows) t.flush(to);
        }
        t.put(place, rows);
    }
    join_moments<V, SAME>(red, d, p, b, share, [&](int g, double mu, float var) {
        const Stat s = finish_stat(mu, var, eps);
        stat[g] = s;
        if (mean != nullptr) {
            mean[(size_t)n * d.G + b.g0 + g] = s.mean;
            rstd[(size_t)n * d.G + b.g0 + g] = s.r;
        }
    });
    __syncthreads();
    if (in) {
        Column<V> col;
        load_column<V>(col, stat, gamma, beta, d, p, b, cv);
        const DropKey key = drop.on ? drop_key(drop) : DropKey{};
#pragma unroll 2
        for (int r = rt; r < r1; r += p.rt)
            write_vector<T, V>(load_raw<T, V>(own + r * pitch), col, act, drop, key, at + (size_t)r * d.C, y);
    }
}

// ---- forward, two passes ----------------------------------------------------------------------------------------------

constexpr int kRing = 8, kBackRing = 4;    // rows that are on their way at a time
constexpr int kBackRun = 64;               // rows that a thread adds up in fp32

template <typename T, int V, bool SAME>
__global__ void __launch_bounds__(kNormThreads, 4)
norm_sums_kernel(const T* __restrict__ x, NormDims d, NormPlan p, double2* __restrict__ part) {
    extern __shared__ uint4 space[];                            // the ring, then [rt][tx] or [rt][tx * V]
    Part* red = space_at<Part>(space, norm_ring_bytes<T, V, 1, kRing>());
    const int n = p.by_blocks(blockIdx.x), split = blockIdx.y;
    const NormBlock b = norm_block<V>(d, p, blockIdx.x - n * p.blocks);
    const int rt = p.by_tx(threadIdx.x), cv = threadIdx.x - rt * p.tx;
    const NormRows share = norm_rows(d, p, split);
    if (rt < p.rt && cv < b.nvec) {
        const int first = split * p.rt + rt, rows = rows_of(share, rt);
        const T* const at[1] = {x + ((size_t)n * d.L) * d.C + b.c0 + cv * V};
        NormStream<T, V, 1, kRing> stream(space, at, first, d.L, p.splits * p.rt, d.C);
        grid_let_go();
        Part* place = moments_at<V, SAME>(red, p, rt, cv);
        Moments<V, SAME> t(place);
        t.start(load_lanes<T, V>(at[0] + (size_t)first * d.C));
        for (int r = 0, run = kFirstRun; r < rows; run = kRun) {
            const int to = min(rows, r + run);
            stream.template run<true>(to - r, [&](int, const Raw<T, V>(&v)[1]) { t.add(lanes_of<T, V>(v[0])); });
            if (to < rows) t.flush(to);
            r = to;
        }
        t.put(place, rows);
    }
    join_moments<V, SAME>(red, d, p, b, share, [&](int g, double mu, float var) {
        part[(((size_t)n * p.splits + split) * d.G + b.g0 + g) * p.pieces + b.piece] = make_double2(mu, var);
    });
}

// Mean and variance of a group from those of the CTAs that share its rows and of its pieces, about the first one's mean; in all lanes.
__device__ __forceinline__ double2 join_parts(const double2* part, const NormDims& d, const NormPlan& p, int n, int g) {
    const double ref = __ldcg(&part[((size_t)n * p.splits * d.G + g) * p.pieces].x);
    const int threads = p.splits * p.rt, base = d.L / threads, more = d.L - base * threads;
    double a = 0.0, q = 0.0;
    for (int k = threadIdx.x & 31; k < p.splits * p.pieces; k += 32) {
        const int s = k / p.pieces, piece = k - s * p.pieces;
        const double2 v = __ldcg(part + (((size_t)n * p.splits + s) * d.G + g) * p.pieces + piece);
        const int rows = base * p.rt + min(max(more - s * p.rt, 0), p.rt), width = p.pieces == 1 ? d.Cg : min(p.piece, d.Cg / p.V - piece * p.piece) * p.V;
        const double weight = (double)rows * (double)width * d.inv_m, e = v.x - ref;
        a += weight * e;
        q += weight * (v.y + e * e);
    }
    a = warp_sum(a);
    q = warp_sum(q);
    return make_double2(ref + a, q - a * a);
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 4)
norm_apply_kernel(const T* __restrict__ x, Param gamma, Param beta, const double2* __restrict__ part, NormDims d, NormPlan p, double eps, int act,
                  Drop drop, T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
    extern __shared__ uint4 space[];                            // the ring, then the groups' mean and 1 / deviation
    Stat* stat = space_at<Stat>(space, norm_ring_bytes<T, V, 1, kRing>());
    const int last = gridDim.x - 1 - blockIdx.x, n = p.by_blocks(last), split = p.splits - 1 - blockIdx.y;
    const NormBlock b = norm_block<V>(d, p, last - n * p.blocks);
    const int rt = p.by_tx(threadIdx.x), cv = threadIdx.x - rt * p.tx;
    const bool in = rt < p.rt && cv < b.nvec;
    const size_t at = ((size_t)n * d.L) * d.C + b.c0 + cv * V;
    const T* const from[1] = {x + at};
    NormStream<T, V, 1, kRing> stream(space, from, split * p.rt + rt, in ? d.L : 0, p.splits * p.rt, d.C);
    grid_wait();
    for (int g = threadIdx.x >> 5; g < b.ng; g += kNormThreads / 32) {
        const double2 v = join_parts(part, d, p, n, b.g0 + g);
        if ((threadIdx.x & 31) == 0) {
            const Stat f = finish_stat(v.x, v.y, eps);
            stat[g] = f;
            if (split == 0 && b.piece == 0 && mean != nullptr) {
                mean[(size_t)n * d.G + b.g0 + g] = f.mean;
                rstd[(size_t)n * d.G + b.g0 + g] = f.r;
            }
        }
    }
    __syncthreads();
    if (!in) return;
    Column<V> col;
    load_column<V>(col, stat, gamma, beta, d, p, b, cv);
    const DropKey key = drop.on ? drop_key(drop) : DropKey{};
    stream.run_all([&](int r, const Raw<T, V>(&v)[1]) { write_vector<T, V>(v[0], col, act, drop, key, at + (size_t)r * d.C, y); });
}

// ---- backward -----------------------------------------------------------------------------------------------------

// The two sums of a group over the CTAs that share its rows and over its pieces, in all lanes.
__device__ __forceinline__ double2 add_parts(const double2* part, const NormDims& d, const NormPlan& p, int n, int g) {
    double a = 0.0, e = 0.0;
    for (int k = threadIdx.x & 31; k < p.splits * p.pieces; k += 32) {
        const int s = k / p.pieces, piece = k - s * p.pieces;
        const double2 v = __ldcg(part + (((size_t)n * p.splits + s) * d.G + g) * p.pieces + piece);
        a += v.x;
        e += v.y;
    }
    return make_double2(warp_sum(a) * d.inv_m, warp_sum(e) * d.inv_m);
}

// What a thread's column needs for u = (x + m) a + o, and for dx = a du + ra + (x + m) rb; m as above.
template <int V> struct BackColumn {
    Lanes<V> m, a, o;
    float r[V];
};
template <int V>
__device__ __forceinline__ void load_back_column(BackColumn<V>& k, const float* mean, const float* rstd, const Param& gamma, const Param& beta,
                                                 const NormDims& d, const NormPlan& p, const NormBlock& b, int n, int cv) {
    int g[V];
    groups_of<V>(d, p, cv * V, g);
    float m[V], a[V], o[V];
    load_params<V>(gamma, b.c0 + cv * V, a);
    load_params<V>(beta, b.c0 + cv * V, o);
    mean += (size_t)n * d.G + b.g0;
    rstd += (size_t)n * d.G + b.g0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        m[j] = -__ldg(mean + g[j]);
        k.r[j] = __ldg(rstd + g[j]);
        a[j] *= k.r[j];
    }
    k.m.set(m);
    k.a.set(a);
    k.o.set(o);
}

// du of V elements (the gradient at u) from that at y, which has been dropped already, and x - mean
template <typename T, int V>
__device__ __forceinline__ void back_du(const Raw<T, V>& xv, const BackColumn<V>& k, int act, Lanes<V>& du, Lanes<V>& e) {
    e = add(lanes_of<T, V>(xv), k.m);
    if (act != LINF_ACT_IDENTITY) du = mul(du, slope<sizeof(T) == 4, V>(fma(e, k.a, k.o), act));
}
template <typename T, int V>
__device__ __forceinline__ void back_du(const Raw<T, V>& xv, const Raw<T, V>& gv, const BackColumn<V>& k, int act, const Drop& drop, const DropKey& key,
                                        size_t i, Lanes<V>& du, Lanes<V>& e) {
    du = lanes_of<T, V>(gv);
    if (drop.on) du = linf::drop<V>(drop, key, i, du);
    back_du<T, V>(xv, k, act, du, e);
}

// Sums of gamma du and gamma du h over each group of the block from its channels' sums (du, du h), which `sums` holds by channel.
template <typename Pair, typename Done>
__device__ __forceinline__ void group_sums(const Pair* sums, const Param& gamma, const NormDims& d, const NormPlan& p, const NormBlock& b, Done done) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int per = p.pieces == 1 ? d.Cg : b.nvec * p.V;
    int wide = 1;                                               // as many lanes to a group as it has channels, up to a warp
    while (wide < per && wide < 32) wide *= 2;
    for (int g0 = (threadIdx.x >> 5) * (32 / wide); g0 < b.ng; g0 += warps * (32 / wide)) {
        const int g = g0 + lane / wide, first = g < b.ng ? lane & (wide - 1) : per;
        double s = 0.0, t = 0.0;
        for (int c = first; c < per; c += wide) {
            const float w = load_param(gamma, b.c0 + g * per + c);
            const Pair v = sums[g * per + c];
            s += (double)w * v.x;
            t += (double)w * v.y;
        }
        for (int o = 1; o < wide; o *= 2) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            t += __shfl_xor_sync(0xffffffffu, t, o);
        }
        if (g < b.ng && (lane & (wide - 1)) == 0) done(g, make_double2(s, t));
    }
}

// Adds the threads' channel sums up along the rows; they end in red's first row.
template <typename Pair> __device__ __forceinline__ void fold_rows(Pair* red, int width, int rt) {
    by_columns(width, rt, [&](int c, int first, int step, auto join) {
        Pair t;
        t.x = t.y = 0;
        for (int r = first; r < rt; r += step) { const Pair v = red[r * width + c]; t.x += v.x; t.y += v.y; }
        if (join(t.x, t.y)) red[c] = t;
    });
}

// ra, rb of a thread's column
template <int V> struct Means { Lanes<V> ra, rb; };
template <int V>
__device__ __forceinline__ void load_means(const float2* stat, const NormDims& d, const NormPlan& p, int cv, const BackColumn<V>& k, Means<V>& m) {
    int g[V];
    groups_of<V>(d, p, cv * V, g);
    float ra[V], rb[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float2 s = stat[g[j]];
        ra[j] = -k.r[j] * s.x;
        rb[j] = -k.r[j] * k.r[j] * s.y;
    }
    m.ra.set(ra);
    m.rb.set(rb);
}
// dx of V elements from du and x - mean
template <typename T, int V>
__device__ __forceinline__ void write_dx(const Lanes<V>& du, const Lanes<V>& e, const BackColumn<V>& k, const Means<V>& m, T* to) {
    store_once<T, V>(to, raw_of<T, V>(fma(e, m.rb, fma(k.a, du, m.ra))));
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 2)
norm_back_kept_kernel(const T* __restrict__ dy, const T* __restrict__ x, Param gamma, Param beta, const float* __restrict__ mean,
                      const float* __restrict__ rstd, NormDims d, NormPlan p, KeptSpace sp, int act, Drop drop, T* __restrict__ dx,
                      float2* __restrict__ by_channel) {
    extern __shared__ uint4 space[];
    T* data = reinterpret_cast<T*>(space);
    float2* red = space_at<float2>(space, sp.red);
    float2* stat = space_at<float2>(space, sp.stat);
    unsigned char* kept = space_at<unsigned char>(space, sp.mask);
    const int chunk = p.by_blocks(blockIdx.x);
    const NormBlock b = norm_block<V>(d, p, blockIdx.x - chunk * p.blocks);
    const int rt = p.by_tx(threadIdx.x), cv = threadIdx.x - rt * p.tx;
    const bool in = rt < p.rt && cv < b.nvec;
    const int r1 = in ? d.L : 0, pitch = p.tx * V;
    T* own = data + cv * V;                                     // x, and behind its rows dy
    T* own_g = own + (size_t)p.rows * pitch;
    const int n1 = min(d.N, (chunk + 1) * p.per_cta);
    const DropKey key = drop.on ? drop_key(drop) : DropKey{};
    float2 total[V];                                            // of all samples of this CTA
#pragma unroll
    for (int j = 0; j < V; ++j) total[j] = make_float2(0.f, 0.f);
    for (int n = chunk * p.per_cta; n < n1; ++n) {
        const size_t at = ((size_t)n * d.L) * d.C + b.c0 + cv * V;
        for (int r = rt; r < r1; r += p.rt) {
            keep_vector<T, V>(own + r * pitch, x + at + (size_t)r * d.C);
            keep_vector<T, V>(own_g + r * pitch, dy + at + (size_t)r * d.C);
        }
        BackColumn<V> col;
        if (in) load_back_column<V>(col, mean, rstd, gamma, beta, d, p, b, n, cv);
        Lanes<V> sum_a = filled<V>(0.f), sum_b = sum_a;
        keep_wait();
        auto sum_row = [&](int r) {
            Lanes<V> du = load_lanes<T, V>(own_g + r * pitch), e;
            if (drop.on) {
                const unsigned mask = drop_mask<V>(drop, key, at + (size_t)r * d.C);
                if (sizeof(T) == 2) kept[r * p.tx + cv] = (unsigned char)mask;
                du = drop_masked<V>(drop, mask, du);
            }
            back_du<T, V>(load_raw<T, V>(own + r * pitch), col, act, du, e);
            sum_a = add(sum_a, du);
            sum_b = fma(du, e, sum_b);
            // fp32: du takes the place of dy; 16-bit types would round it, and work it out again
            if (sizeof(T) == 4) *reinterpret_cast<Raw<T, V>*>(own_g + r * pitch) = raw_of<T, V>(du);
        };
        if constexpr (V == 1 && sizeof(T) == 2) {               // up to 127 rows to a thread (else 63): in runs, which are added up
            for (int r0 = rt; r0 < r1; r0 += 32 * p.rt) {
                const Lanes<V> a = sum_a, b = sum_b;
                sum_a = sum_b = filled<V>(0.f);
#pragma unroll 2
                for (int r = r0; r < min(r0 + 32 * p.rt, r1); r += p.rt) sum_row(r);
                sum_a = add(a, sum_a);
                sum_b = add(b, sum_b);
            }
        } else {
#pragma unroll 2
            for (int r = rt; r < r1; r += p.rt) sum_row(r);
        }
        float sa[V], sb[V];
        sum_a.get(sa);
        sum_b.get(sb);
        if (in) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                sb[j] *= col.r[j];
                total[j].x += sa[j];
                total[j].y += sb[j];
            }
        }
        if (dx == nullptr) continue;                            // the same for every thread
        if (rt < p.rt) {
#pragma unroll
            for (int j = 0; j < V; ++j) red[rt * pitch + cv * V + j] = make_float2(sa[j], sb[j]);
        }
        __syncthreads();
        if (p.rt > 1) {
            fold_rows(red, pitch, p.rt);
            __syncthreads();
        }
        group_sums(red, gamma, d, p, b, [&](int g, double2 v) { stat[g] = make_float2((float)(v.x * d.inv_m), (float)(v.y * d.inv_m)); });
        __syncthreads();
        if (in) {
            Means<V> means;
            load_means<V>(stat, d, p, cv, col, means);
#pragma unroll 2
            for (int r = rt; r < r1; r += p.rt) {
                Lanes<V> du = load_lanes<T, V>(own_g + r * pitch), e;
                if (sizeof(T) == 4) {
                    e = add(load_lanes<T, V>(own + r * pitch), col.m);
                } else {
                    if (drop.on) du = drop_masked<V>(drop, kept[r * p.tx + cv], du);
                    back_du<T, V>(load_raw<T, V>(own + r * pitch), col, act, du, e);
                }
                write_dx<T, V>(du, e, col, means, dx + at + (size_t)r * d.C);
            }
        }
        __syncthreads();
    }
    if (rt < p.rt) {
#pragma unroll
        for (int j = 0; j < V; ++j) red[rt * pitch + cv * V + j] = total[j];
    }
    __syncthreads();
    fold_rows(red, pitch, p.rt);
    __syncthreads();
    for (int c = threadIdx.x; c < b.nvec * V; c += blockDim.x) by_channel[(size_t)chunk * d.C + b.c0 + c] = red[c];
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 2)
norm_back_sums_kernel(const T* __restrict__ dy, const T* __restrict__ x, Param gamma, Param beta, const float* __restrict__ mean,
                      const float* __restrict__ rstd, NormDims d, NormPlan p, int act, Drop drop, float2* __restrict__ by_channel,
                      double2* __restrict__ by_group) {
    extern __shared__ uint4 space[];                            // the ring, then [rt][tx * V]
    double2* red = space_at<double2>(space, norm_ring_bytes<T, V, 2, kBackRing>());
    const int n = p.by_blocks(blockIdx.x), split = blockIdx.y;
    const NormBlock b = norm_block<V>(d, p, blockIdx.x - n * p.blocks);
    const int rt = p.by_tx(threadIdx.x), cv = threadIdx.x - rt * p.tx;
    const int width = p.tx * V;
    // fp32 over a run of rows, 64-bit over the runs where there is more than one (the sums kernel of 16 x 128 x 160 x 160 bf16: 68 us, with 64-bit
    // pairs in any case 72)
    const NormRows share = norm_rows(d, p, split);
    const bool one = share.base + (share.more > 0 ? 1 : 0) <= kBackRun;
    if (rt < p.rt && cv < b.nvec) {
        Lanes<V> sum_a = filled<V>(0.f), sum_b = sum_a;
        BackColumn<V> col;
        const size_t at = ((size_t)n * d.L) * d.C + b.c0 + cv * V;
        const T* const from[2] = {x + at, dy + at};
        NormStream<T, V, 2, kBackRing> stream(space, from, split * p.rt + rt, d.L, p.splits * p.rt, d.C);
        const int rows = rows_of(share, rt);
        grid_let_go();
        load_back_column<V>(col, mean, rstd, gamma, beta, d, p, b, n, cv);
        const DropKey key = drop.on ? drop_key(drop) : DropKey{};
        // into the thread's pairs: V sums of du and of du h
        auto put = [&](auto* own, bool begun) {
            float sa[V], sb[V];
            sum_a.get(sa);
            sum_b.get(sb);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                auto v = own[j];
                v.x = (begun ? v.x : 0) + sa[j];
                v.y = (begun ? v.y : 0) + sb[j] * col.r[j];
                own[j] = v;
            }
        };
        for (int left = rows, run = 0; left > 0; left -= kBackRun, ++run) {
            stream.template run<false>(min(left, kBackRun), [&](int r, const Raw<T, V>(&v)[2]) {
                Lanes<V> du, e;
                back_du<T, V>(v[0], v[1], col, act, drop, key, at + (size_t)r * d.C, du, e);
                sum_a = add(sum_a, du);
                sum_b = fma(du, e, sum_b);
            });
            if (one) break;
            put(red + rt * width + cv * V, run > 0);
            sum_a = sum_b = filled<V>(0.f);
        }
        if (one) put(reinterpret_cast<float2*>(red) + rt * width + cv * V, false);
    }
    auto finish = [&](auto* pairs) {
        __syncthreads();
        fold_rows(pairs, width, p.rt);
        __syncthreads();
        for (int c = threadIdx.x; c < b.nvec * V; c += kNormThreads)
            by_channel[((size_t)n * p.splits + split) * d.C + b.c0 + c] = make_float2((float)pairs[c].x, (float)pairs[c].y);
        group_sums(pairs, gamma, d, p, b,
                   [&](int g, double2 v) { by_group[(((size_t)n * p.splits + split) * d.G + b.g0 + g) * p.pieces + b.piece] = v; });
    };
    if (one) finish(reinterpret_cast<float2*>(red));
    else finish(red);
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 2)
norm_back_apply_kernel(const T* __restrict__ dy, const T* __restrict__ x, Param gamma, Param beta, const float* __restrict__ mean,
                       const float* __restrict__ rstd, NormDims d, NormPlan p, int act, Drop drop, const double2* __restrict__ by_group,
                       T* __restrict__ dx) {
    extern __shared__ uint4 space[];                            // the ring, then the groups' two means
    float2* stat = space_at<float2>(space, norm_ring_bytes<T, V, 2, kBackRing>());
    const int last = gridDim.x - 1 - blockIdx.x, n = p.by_blocks(last), split = p.splits - 1 - blockIdx.y;
    const NormBlock b = norm_block<V>(d, p, last - n * p.blocks);
    const int rt = p.by_tx(threadIdx.x), cv = threadIdx.x - rt * p.tx;
    const bool in = rt < p.rt && cv < b.nvec;
    const size_t at = ((size_t)n * d.L) * d.C + b.c0 + cv * V;
    const T* const from[2] = {x + at, dy + at};
    NormStream<T, V, 2, kBackRing> stream(space, from, split * p.rt + rt, in ? d.L : 0, p.splits * p.rt, d.C);
    grid_wait();
    for (int g = threadIdx.x >> 5; g < b.ng; g += kNormThreads / 32) {
        const double2 v = add_parts(by_group, d, p, n, b.g0 + g);
        if ((threadIdx.x & 31) == 0) stat[g] = make_float2((float)v.x, (float)v.y);
    }
    __syncthreads();
    if (!in) return;
    BackColumn<V> col;
    load_back_column<V>(col, mean, rstd, gamma, beta, d, p, b, n, cv);
    Means<V> means;
    load_means<V>(stat, d, p, cv, col, means);
    const DropKey key = drop.on ? drop_key(drop) : DropKey{};
    stream.run_all([&](int r, const Raw<T, V>(&v)[2]) {
        const size_t i = at + (size_t)r * d.C;
        Lanes<V> du, e;
        back_du<T, V>(v[0], v[1], col, act, drop, key, i, du, e);
        write_dx<T, V>(du, e, col, means, dx + i);
    });
}

// dgamma, dbeta: the rows of per-channel sums in 64 bits, 8 channels to a CTA (a row's piece is two sectors).  A thread has 8 rows on their way
// at a time: with few CTAs the time is the latency of its loads.
constexpr int kParamThreads = 512, kParamRows = kParamThreads / 8, kParamLoads = 8;
__global__ void __launch_bounds__(kParamThreads)
norm_params_kernel(const float2* __restrict__ by_channel, long long count, int C, void* __restrict__ dgamma, void* __restrict__ dbeta, int ptype) {
    __shared__ double2 red[kParamThreads / 32][8];
    const int col = threadIdx.x & 7, lane = threadIdx.x >> 3, c = blockIdx.x * 8 + col;
    double a = 0.0, e = 0.0;
    grid_wait();
    if (c < C) {
        for (long long k0 = lane; k0 < count; k0 += kParamRows * kParamLoads) {
            float2 v[kParamLoads];
#pragma unroll
            for (int u = 0; u < kParamLoads; ++u) {
                const long long k = k0 + u * kParamRows;
                v[u] = k < count ? __ldcg(by_channel + k * C + c) : make_float2(0.f, 0.f);
            }
#pragma unroll
            for (int u = 0; u < kParamLoads; ++u) { a += v[u].x; e += v[u].y; }
        }
    }
#pragma unroll
    for (int o = 8; o < 32; o *= 2) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        e += __shfl_xor_sync(0xffffffffu, e, o);
    }
    if ((threadIdx.x & 31) < 8) red[threadIdx.x >> 5][col] = make_double2(a, e);
    __syncthreads();
    if (threadIdx.x >= 8 || c >= C) return;
#pragma unroll
    for (int k = 1; k < kParamThreads / 32; ++k) { a += red[k][col].x; e += red[k][col].y; }
    if (dbeta != nullptr) store_param(dbeta, c, ptype, (float)a);
    if (dgamma != nullptr) store_param(dgamma, c, ptype, (float)e);
}

// ---- launches -----------------------------------------------------------------------------------------------------

NormKind forward_kind(int type) { return {type == LINF_F32 ? 4 : 2, 1, false}; }
NormKind backward_kind(int type) { return {type == LINF_F32 ? 4 : 2, 2, true}; }

// The workspace of a call: forward, two passes: the parts; backward: the channels' sums, and the parts of two passes.
size_t parts_bytes(const NormDims& d, const NormPlan& p) { return p.kept ? 0 : sizeof(double2) * (size_t)d.N * p.splits * d.G * p.pieces; }
long long channel_rows(const NormPlan& p) { return (long long)p.chunks * p.splits; }
constexpr int kDenseCtas = 8, kDenseBackCtas = 3;      // of each SM
size_t dense_workspace(const NormDims& d, const DensePlan& p) { return sizeof(float2) * (size_t)p.chunks * p.subs * d.C; }
size_t workspace(const NormDims& d, const NormPlan& p, bool back) {
    return parts_bytes(d, p) + (back ? sizeof(float2) * (size_t)channel_rows(p) * d.C : 0);
}

template <typename T, int V, bool SAME>
int forward_as(const T* x, const NormGiven& given, const NormDims& d, const NormPlan& p, double eps, int act, const Drop& drop, T* y, float* mean,
               float* rstd, void* ws, cudaStream_t st) {
    if (p.kept) {
        const KeptSpace sp = kept_space(p, sizeof(T), 1, sizeof(Part), SAME, sizeof(Stat), false);
        return launch_kept<norm_kept_kernel<T, V, SAME>>(p, sp.bytes, st, x, given.gamma, given.beta, d, p, sp, eps, act, drop, y, mean, rstd);
    }
    const dim3 grid((unsigned)(p.blocks * d.N), p.splits);
    double2* part = static_cast<double2*>(ws);
    const size_t ring = norm_ring_bytes<T, V, 1, kRing>();
    const size_t one = ring + sizeof(Part) * p.rt * p.tx * (SAME ? 1 : V), two = ring + sizeof(Stat) * p.groups;
    if (!allow_shared<norm_sums_kernel<T, V, SAME>>(one) || !allow_shared<norm_apply_kernel<T, V>>(two)) return LINF_ERR_LAUNCH;
    norm_sums_kernel<T, V, SAME><<<grid, kNormThreads, one, st>>>(x, d, p, part);
    if (launch_status()) return LINF_ERR_LAUNCH;
    return launch_behind(norm_apply_kernel<T, V>, grid, kNormThreads, two, st, x, given.gamma, given.beta, part, d, p, eps, act, drop, y, mean, rstd);
}
template <typename T, int V>
int forward(const T* x, const NormGiven& given, const NormDims& d, const NormPlan& p, double eps, int act, const Drop& drop, T* y, float* mean,
            float* rstd, void* ws, cudaStream_t st) {
    if constexpr (V > 1)
        if (!p.same) return forward_as<T, V, false>(x, given, d, p, eps, act, drop, y, mean, rstd, ws, st);
    return forward_as<T, V, true>(x, given, d, p, eps, act, drop, y, mean, rstd, ws, st);
}

template <typename T, int V>
int backward(const T* dy, const T* x, const NormGiven& given, int ptype, const float* mean, const float* rstd, const NormDims& d, const NormPlan& p,
             int act, const Drop& drop, T* dx, void* dgamma, void* dbeta, void* ws, cudaStream_t st) {
    double2* by_group = static_cast<double2*>(ws);
    float2* by_channel = reinterpret_cast<float2*>(static_cast<char*>(ws) + parts_bytes(d, p));
    if (p.kept) {
        const KeptSpace sp = kept_space(p, sizeof(T), 2, sizeof(float2), false, sizeof(float2), drop.on && sizeof(T) == 2);
        const int rc = launch_kept<norm_back_kept_kernel<T, V>>(p, sp.bytes, st, dy, x, given.gamma, given.beta, mean, rstd, d, p, sp, act, drop,
                                   dx, by_channel);
        if (rc) return rc;
    } else {
        const dim3 grid((unsigned)(p.blocks * d.N), p.splits);
        const size_t ring = norm_ring_bytes<T, V, 2, kBackRing>();
        const size_t one = ring + sizeof(double2) * p.rt * p.tx * V, two = ring + sizeof(float2) * p.groups;
        if (!allow_shared<norm_back_sums_kernel<T, V>>(one) || !allow_shared<norm_back_apply_kernel<T, V>>(two)) return LINF_ERR_LAUNCH;
        norm_back_sums_kernel<T, V><<<grid, kNormThreads, one, st>>>(dy, x, given.gamma, given.beta, mean, rstd, d, p, act, drop, by_channel, by_group);
        if (launch_status()) return LINF_ERR_LAUNCH;
        if (dx != nullptr) {
            const int rc = launch_behind(norm_back_apply_kernel<T, V>, grid, kNormThreads, two, st, dy, x, given.gamma, given.beta, mean, rstd, d, p, act,
                                         drop, by_group, dx);
            if (rc) return rc;
        }
    }
    return dgamma != nullptr || dbeta != nullptr ? norm_params(by_channel, channel_rows(p), d.C, dgamma, dbeta, ptype, st) : LINF_OK;
}

}  // namespace

bool norm_given(const void* gamma, const void* beta, int ptype, NormGiven* g) {
    static std::atomic<void*> known[kMaxDevices];
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return false; }
    void* at = dev < kMaxDevices ? known[dev].load(std::memory_order_relaxed) : nullptr;
    if (at == nullptr) {
        if (cudaGetSymbolAddress(&at, g_own) != cudaSuccess) { cudaGetLastError(); return false; }
        if (dev < kMaxDevices) known[dev].store(at, std::memory_order_relaxed);
    }
    Own* own = static_cast<Own*>(at);
    auto given = [&](const void* v, const float* instead) {
        if (v == nullptr) return Param{instead, PARAM_ONE};
        if (ptype == LINF_F32) return Param{v, aligned16(v) ? PARAM_WIDE : PARAM_F32};
        return Param{v, ptype == LINF_F16 ? PARAM_F16 : PARAM_BF16};
    };
    g->gamma = given(gamma, &own->one);
    g->beta = given(beta, &own->zero);
    g->idle = own->rng;
    return true;
}

int norm_params(const float2* by_channel, long long count, int C, void* dgamma, void* dbeta, int ptype, cudaStream_t st) {
    return launch_behind(norm_params_kernel, dim3(norm_param_ctas(C)), kParamThreads, 0, st, by_channel, count, C, dgamma, dbeta, ptype);
}

size_t group_norm_workspace(int N, int C, int G, int L, int type, bool back) {
    // a plan goes by the pointers' alignment; either may run
    size_t most = 0;
    for (int k = 0; k < 2; ++k) {
        NormDims d;
        NormPlan p;
        DensePlan dp;
        if (norm_make(N, C, G, L, back ? backward_kind(type) : forward_kind(type), k == 0, &d, &p) != LINF_OK) return 0;
        const bool dense = dense_plan(d, type == LINF_F32 ? 4 : 2, k == 0, sm_count() * (back ? kDenseBackCtas : kDenseCtas), &dp);
        const size_t need = dense ? (back ? dense_workspace(d, dp) : 0) : workspace(d, p, back);
        if (need > most) most = need;
    }
    return (most + 255) / 256 * 256;
}

#define LINF_BY_VECTOR(CALL16, CALL32)                                                                             \
    switch (type) {                                                                                                \
        case LINF_F32:                                                                                             \
            if (p.V == 4) return CALL32(float, 4);                                                                 \
            if (p.V == 2) return CALL32(float, 2);                                                                 \
            return CALL32(float, 1);                                                                               \
        case LINF_F16:                                                                                             \
            if (p.V == 8) return CALL16(__half, 8);                                                                \
            if (p.V == 4) return CALL16(__half, 4);                                                                \
            if (p.V == 2) return CALL16(__half, 2);                                                                \
            return CALL16(__half, 1);                                                                              \
        default:                                                                                                   \
            if (p.V == 8) return CALL16(__nv_bfloat16, 8);                                                         \
            if (p.V == 4) return CALL16(__nv_bfloat16, 4);                                                         \
            if (p.V == 2) return CALL16(__nv_bfloat16, 2);                                                         \
            return CALL16(__nv_bfloat16, 1);                                                                       \
    }

int group_norm_forward(const void* x, const void* gamma, const void* beta, int N, int C, int G, int L, int type, int ptype, double eps, int act,
                       double rate, const long long* rng, void* y, float* mean, float* rstd, void* ws, size_t ws_bytes, cudaStream_t st) {
    NormDims d;
    NormPlan p;
    const int rc = norm_make(N, C, G, L, forward_kind(type), aligned16(x) && aligned16(y), &d, &p);
    if (rc) return rc;
    DensePlan dp;
    const bool dense = dense_plan(d, type == LINF_F32 ? 4 : 2, aligned16(x) && aligned16(y), sm_count() * kDenseCtas, &dp);
    const size_t need = dense ? 0 : workspace(d, p, false);
    if (need > 0 && (ws == nullptr || !aligned16(ws) || ws_bytes < need)) return LINF_ERR_WORKSPACE;
    NormGiven given;
    if (!norm_given(gamma, beta, ptype, &given)) return LINF_ERR_LAUNCH;
    Drop drop;
    if (!make_drop(rate, rng, given.idle, &drop)) return LINF_ERR_RATE;
    if (dense) return dense_norm_forward(x, given, d, dp, type, eps, act, drop, y, mean, rstd, st);
#define LINF_CALL(T, V) forward<T, V>(static_cast<const T*>(x), given, d, p, eps, act, drop, static_cast<T*>(y), mean, rstd, ws, st)
    LINF_BY_VECTOR(LINF_CALL, LINF_CALL)
#undef LINF_CALL
}

int group_norm_backward(const void* dy, const void* x, const void* gamma, const void* beta, const float* mean, const float* rstd, int N, int C,
                        int G, int L, int type, int ptype, int act, double rate, const long long* rng, void* dx, void* dgamma, void* dbeta,
                        void* ws, size_t ws_bytes, cudaStream_t st) {
    NormDims d;
    NormPlan p;
    const int rc = norm_make(N, C, G, L, backward_kind(type), aligned16(x) && aligned16(dy) && aligned16(dx), &d, &p);
    if (rc) return rc;
    DensePlan dp;
    const bool dense = dense_plan(d, type == LINF_F32 ? 4 : 2, aligned16(x) && aligned16(dy) && aligned16(dx), sm_count() * kDenseBackCtas, &dp);
    if (ws == nullptr || !aligned16(ws) || ws_bytes < (dense ? dense_workspace(d, dp) : workspace(d, p, true))) return LINF_ERR_WORKSPACE;
    NormGiven given;
    if (!norm_given(gamma, beta, ptype, &given)) return LINF_ERR_LAUNCH;
    Drop drop;
    if (!make_drop(rate, rng, given.idle, &drop)) return LINF_ERR_RATE;
    if (dense) {
        float2* by_channel = static_cast<float2*>(ws);
        const int done = dense_norm_backward(dy, x, given, mean, rstd, d, dp, type, act, drop, dx, by_channel, st);
        if (done || (dgamma == nullptr && dbeta == nullptr)) return done;
        return norm_params(by_channel, (long long)dp.chunks * dp.subs, C, dgamma, dbeta, ptype, st);
    }
#define LINF_CALL(T, V)                                                                                                                   \
    backward<T, V>(static_cast<const T*>(dy), static_cast<const T*>(x), given, ptype, mean, rstd, d, p, act, drop, static_cast<T*>(dx), \
                   dgamma, dbeta, ws, st)
    LINF_BY_VECTOR(LINF_CALL, LINF_CALL)
#undef LINF_CALL
}

}  // namespace linf
