// Group norm of dense activations [N, C] (one position): a group is a row of C/G neighbouring values.
//
// As many threads as the row needs (a power of two, from one lane to 512 threads) hold a row in registers: one load, two reductions, one store.  Such a
// slot keeps its group and goes through a range of samples, so that gamma and beta are read once and, in the backward pass, the
// sums for their gradients stay in registers; the next sample's loads are on their way while one is reduced.  Bound by the
// instructions and the latency of the reductions.  Measured on one B200, us, forward / forward and backward: 512 x 5120 fp32, 32 groups, tanh 12.5 /
// -; 2048 x 5120 bf16, 32 groups, tanh 30 / 82; 2048 x 5120 fp32, one group, no activation 40 / 97.  (The kernels for maps, whose CTA begins
// anew for each sample, took 18.6 / -, 58 / 172 and 99 / 345.)
#include "group_norm.cuh"

namespace linf {
namespace {

constexpr int kDenseMost = 512;

// sums of two values over the `tpr` threads of a slot, in all of them; part: two floats for each warp and turn
__device__ __forceinline__ float2 slot_sum(float a, float b, int tpr, float2* part) {
    const int lanes = tpr < 32 ? tpr : 32;
    for (int o = 1; o < lanes; o *= 2) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (tpr <= 32) return make_float2(a, b);
    const int warp = threadIdx.x >> 5, warps = tpr >> 5, first = warp / warps * warps;
    if ((threadIdx.x & 31) == 0) part[warp] = make_float2(a, b);
    __syncthreads();
    float2 t = part[first];
    for (int w = 1; w < warps; ++w) { t.x += part[first + w].x; t.y += part[first + w].y; }
    return t;
}

struct DenseSlot { int g, t, first, iters, n0, n1; bool in; };
__device__ __forceinline__ DenseSlot dense_slot(const NormDims& d, const DensePlan& p) {
    DenseSlot s;
    const int slot = threadIdx.x / p.tpr, sub = slot / p.groups;
    s.t = threadIdx.x - slot * p.tpr;
    s.g = blockIdx.y * p.groups + slot - sub * p.groups;
    s.in = sub < p.subs && s.g < d.G;
    s.n0 = blockIdx.x * p.per;
    s.n1 = min(d.N, s.n0 + p.per);
    s.first = s.n0 + sub;
    s.iters = (s.n1 - s.n0 + p.subs - 1) / p.subs;              // the same for the whole CTA
    return s;
}

template <typename T, int V, int K>
__device__ __forceinline__ void dense_load(const T* row, bool in, int t, int tpr, int vecs, Raw<T, V> (&v)[K]) {
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (in && t + k * tpr < vecs) v[k] = load_once<T, V>(row + (t + k * tpr) * V);
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(kDenseMost)
dense_norm_kernel(const T* __restrict__ x, Param gamma, Param beta, NormDims d, DensePlan p, double eps, int act, Drop drop, T* __restrict__ y,
                  float* __restrict__ mean, float* __restrict__ rstd) {
    __shared__ float2 part[2][kDenseMost / 32];
    const DenseSlot s = dense_slot(d, p);
    const int vecs = d.Cg / V;
    const DropKey key = drop.on ? drop_key(drop) : DropKey{};
    Lanes<V> w[K], o[K];
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (s.in && s.t + k * p.tpr < vecs) {
            float f[V];
            load_params<V>(gamma, s.g * d.Cg + (s.t + k * p.tpr) * V, f);
            w[k].set(f);
            load_params<V>(beta, s.g * d.Cg + (s.t + k * p.tpr) * V, f);
            o[k].set(f);
        }
    const float inv = (float)d.inv_m;
    Raw<T, V> v[K];
    dense_load<T, V, K>(x + ((size_t)s.first * d.G + s.g) * d.Cg, s.in && s.first < s.n1, s.t, p.tpr, vecs, v);
    for (int i = 0; i < s.iters; ++i) {
        const int n = s.first + i * p.subs;
        const bool in = s.in && n < s.n1;
        const size_t row = ((size_t)n * d.G + s.g) * d.Cg;
        Lanes<V> f[K];
        float a = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (in && s.t + k * p.tpr < vecs) {
                f[k] = lanes_of<T, V>(v[k]);
                float e[V];
                f[k].get(e);
#pragma unroll
                for (int j = 0; j < V; ++j) a += e[j];
            }
        }
        dense_load<T, V, K>(x + row + (size_t)p.subs * d.C, s.in && n + p.subs < s.n1, s.t, p.tpr, vecs, v);
        const float mu = slot_sum(a * inv, 0.f, p.tpr, part[0]).x;       // means of a thread's values: neither sum leaves fp32 first
        const Lanes<V> shift = filled<V>(-mu);
        float q = 0.f;
        a = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (in && s.t + k * p.tpr < vecs) {
                f[k] = add(f[k], shift);
                float e[V];
                f[k].get(e);
#pragma unroll
                for (int j = 0; j < V; ++j) { a += e[j]; q = fmaf(e[j], e[j], q); }
            }
        // the values about mu: what the rounding of mu left of their mean is taken off as well
        const float2 m = slot_sum(a * inv, q * inv, p.tpr, part[1]);
        const float rest = m.x, r = 1.f / sqrtf(fmaxf(fmaf(-rest, rest, m.y), 0.f) + (m.y != m.y ? m.y : (float)eps));
        if (!in) continue;
        if (s.t == 0 && mean != nullptr) {
            mean[(size_t)n * d.G + s.g] = mu + rest;
            rstd[(size_t)n * d.G + s.g] = r;
        }
        const Lanes<V> scale = filled<V>(r), left = filled<V>(-rest);
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (s.t + k * p.tpr < vecs) {
                const size_t at = row + (s.t + k * p.tpr) * V;
                Lanes<V> u = activate<sizeof(T) == 4, V>(fma(mul(add(f[k], left), scale), w[k], o[k]), act);
                if (drop.on) u = linf::drop<V>(drop, key, at, u);
                store_once<T, V>(y + at, raw_of<T, V>(u));
            }
    }
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(kDenseMost)
dense_norm_back_kernel(const T* __restrict__ dy, const T* __restrict__ x, Param gamma, Param beta, const float* __restrict__ mean,
                       const float* __restrict__ rstd, NormDims d, DensePlan p, int act, Drop drop, T* __restrict__ dx, float2* __restrict__ by_channel) {
    __shared__ float2 part[2][kDenseMost / 32];
    const DenseSlot s = dense_slot(d, p);
    const int vecs = d.Cg / V;
    const DropKey key = drop.on ? drop_key(drop) : DropKey{};
    Lanes<V> w[K], o[K], sum_a[K], sum_b[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        sum_a[k] = sum_b[k] = filled<V>(0.f);
        if (s.in && s.t + k * p.tpr < vecs) {
            float f[V];
            load_params<V>(gamma, s.g * d.Cg + (s.t + k * p.tpr) * V, f);
            w[k].set(f);
            load_params<V>(beta, s.g * d.Cg + (s.t + k * p.tpr) * V, f);
            o[k].set(f);
        }
    }
    const float inv = (float)d.inv_m;
    Raw<T, V> v[K], g[K];
    dense_load<T, V, K>(x + ((size_t)s.first * d.G + s.g) * d.Cg, s.in && s.first < s.n1, s.t, p.tpr, vecs, v);
    dense_load<T, V, K>(dy + ((size_t)s.first * d.G + s.g) * d.Cg, s.in && s.first < s.n1, s.t, p.tpr, vecs, g);
    for (int i = 0; i < s.iters; ++i) {
        const int n = s.first + i * p.subs;
        const bool in = s.in && n < s.n1;
        const size_t row = ((size_t)n * d.G + s.g) * d.Cg;
        const float mu = in ? __ldg(mean + (size_t)n * d.G + s.g) : 0.f, r = in ? __ldg(rstd + (size_t)n * d.G + s.g) : 0.f;
        const Lanes<V> shift = filled<V>(-mu), scale = filled<V>(r);
        Lanes<V> du[K], h[K];
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (in && s.t + k * p.tpr < vecs) {
                h[k] = mul(add(lanes_of<T, V>(v[k]), shift), scale);
                du[k] = lanes_of<T, V>(g[k]);
                if (drop.on) du[k] = linf::drop<V>(drop, key, row + (s.t + k * p.tpr) * V, du[k]);
                if (act != LINF_ACT_IDENTITY) du[k] = mul(du[k], slope<sizeof(T) == 4, V>(fma(h[k], w[k], o[k]), act));
                sum_a[k] = add(sum_a[k], du[k]);
                sum_b[k] = fma(du[k], h[k], sum_b[k]);
                du[k] = mul(du[k], w[k]);                        // gamma du from here on
                float f[V], e[V];
                du[k].get(f);
                mul(du[k], h[k]).get(e);
#pragma unroll
                for (int j = 0; j < V; ++j) { a += f[j]; b += e[j]; }
            }
        dense_load<T, V, K>(x + row + (size_t)p.subs * d.C, s.in && n + p.subs < s.n1, s.t, p.tpr, vecs, v);
        dense_load<T, V, K>(dy + row + (size_t)p.subs * d.C, s.in && n + p.subs < s.n1, s.t, p.tpr, vecs, g);
        if (dx == nullptr) continue;                            // the same for every thread
        const float2 m = slot_sum(a, b, p.tpr, part[i & 1]);
        if (!in) continue;
        const Lanes<V> ma = filled<V>(-m.x * inv), mb = filled<V>(-m.y * inv);
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (s.t + k * p.tpr < vecs)
                store_once<T, V>(dx + row + (s.t + k * p.tpr) * V, raw_of<T, V>(mul(fma(h[k], mb, add(du[k], ma)), scale)));
    }
    if (!s.in) return;
    float2* to = by_channel + ((size_t)blockIdx.x * p.subs + (s.first - s.n0)) * d.C + s.g * d.Cg;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (s.t + k * p.tpr < vecs) {
            float a[V], b[V];
            sum_a[k].get(a);
            sum_b[k].get(b);
#pragma unroll
            for (int j = 0; j < V; ++j) to[(s.t + k * p.tpr) * V + j] = make_float2(a[j], b[j]);
        }
}

template <int V> struct DenseK { static constexpr int value = V == 8 ? 2 : 4; };

}  // namespace

// Whether a slot can hold a row; its plan.  ctas: CTAs that the call should have at least, as far as there are samples; a slot takes
// kDenseSamples of them at most, whose sums for the parameters' gradients it adds up in fp32.
bool dense_plan(const NormDims& d, int elem_bytes, bool aligned, int ctas, DensePlan* p) {
    if (d.L != 1) return false;
    const int widths[4] = {16 / elem_bytes, 8 / elem_bytes, 4 / elem_bytes, 1};
    for (int k = 0; k < 4; ++k) {
        const int V = widths[k];
        if (V > 1 && (!aligned || d.Cg % V != 0)) continue;
        p->V = V;
        break;
    }
    const int vecs = d.Cg / p->V, keep = p->V == 8 ? 2 : 4;
    p->tpr = 1;
    while (p->tpr <= kDenseMost && p->tpr * keep < vecs) p->tpr *= 2;
    if (p->tpr > kDenseMost) return false;
    p->threads = p->tpr > kNormThreads ? p->tpr : kNormThreads;
    const int slots = p->threads / p->tpr;
    p->groups = d.G < slots ? d.G : slots;
    p->subs = slots / p->groups;
    p->blocks = norm_ceil(d.G, p->groups);
    if (p->blocks > 65535) return false;
    long long chunks = norm_ceil(ctas, p->blocks);
    if (chunks > norm_ceil(d.N, p->subs)) chunks = norm_ceil(d.N, p->subs);
    if (chunks < norm_ceil(d.N, (long long)p->subs * kDenseSamples)) chunks = norm_ceil(d.N, (long long)p->subs * kDenseSamples);
    p->per = norm_ceil(d.N, chunks);
    p->chunks = norm_ceil(d.N, p->per);
    return true;
}

#define LINF_DENSE(CALL)                                                              \
    switch (type) {                                                                   \
        case LINF_F32:                                                                \
            if (p.V == 4) return CALL(float, 4);                                      \
            if (p.V == 2) return CALL(float, 2);                                      \
            return CALL(float, 1);                                                    \
        case LINF_F16:                                                                \
            if (p.V == 8) return CALL(__half, 8);                                     \
            if (p.V == 4) return CALL(__half, 4);                                     \
            if (p.V == 2) return CALL(__half, 2);                                     \
            return CALL(__half, 1);                                                   \
        default:                                                                      \
            if (p.V == 8) return CALL(__nv_bfloat16, 8);                              \
            if (p.V == 4) return CALL(__nv_bfloat16, 4);                              \
            if (p.V == 2) return CALL(__nv_bfloat16, 2);                              \
            return CALL(__nv_bfloat16, 1);                                            \
    }

namespace {
template <typename T, int V>
int go_forward(const void* x, const NormGiven& given, const NormDims& d, const DensePlan& p, double eps, int act, const Drop& drop, void* y, float* mean,
               float* rstd, cudaStream_t st) {
    const auto kernel = dense_norm_kernel<T, V, DenseK<V>::value>;
    const dim3 grid(p.chunks, p.blocks);
    kernel<<<grid, p.threads, 0, st>>>(static_cast<const T*>(x), given.gamma, given.beta, d, p, eps, act, drop, static_cast<T*>(y), mean, rstd);
    return launch_status();
}
template <typename T, int V>
int go_backward(const void* dy, const void* x, const NormGiven& given, const float* mean, const float* rstd, const NormDims& d, const DensePlan& p, int act,
                const Drop& drop, void* dx, float2* by_channel, cudaStream_t st) {
    const auto kernel = dense_norm_back_kernel<T, V, DenseK<V>::value>;
    const dim3 grid(p.chunks, p.blocks);
    kernel<<<grid, p.threads, 0, st>>>(static_cast<const T*>(dy), static_cast<const T*>(x), given.gamma, given.beta, mean, rstd, d, p, act, drop,
                                       static_cast<T*>(dx), by_channel);
    return launch_status();
}
}  // namespace

int dense_norm_forward(const void* x, const NormGiven& given, const NormDims& d, const DensePlan& p, int type, double eps, int act, const Drop& drop,
                       void* y, float* mean, float* rstd, cudaStream_t st) {
#define LINF_CALL(T, V) go_forward<T, V>(x, given, d, p, eps, act, drop, y, mean, rstd, st)
    LINF_DENSE(LINF_CALL)
#undef LINF_CALL
}

int dense_norm_backward(const void* dy, const void* x, const NormGiven& given, const float* mean, const float* rstd, const NormDims& d, const DensePlan& p,
                        int type, int act, const Drop& drop, void* dx, float2* by_channel, cudaStream_t st) {
#define LINF_CALL(T, V) go_backward<T, V>(dy, x, given, mean, rstd, d, p, act, drop, dx, by_channel, st)
    LINF_DENSE(LINF_CALL)
#undef LINF_CALL
}

}  // namespace linf
