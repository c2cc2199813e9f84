// How the group-norm kernels deal a [N, L, C] activation (channels last) out to CTAs.
//
// A CTA works on a column block -- some whole groups, or a piece of one group -- of a range of rows (positions) of one sample.
// Its threads form `rt` rows of `tx` vectors; a thread keeps its column, so that parameters and per-channel sums stay in registers.
// Vectors are as wide as C, the groups and the pointers' alignment allow: a block of whole groups starts and ends on a vector.
//
// Where a CTA's shared memory holds a sample's column block, the CTA keeps it there ("kept"): every tensor is read once, reduced and
// written.  What is larger takes two passes over memory: sums of parts of the rows, then, in a second launch whose CTAs add those up first and
// which takes the samples in the opposite order, the results: what was read last is still in L2.
#pragma once

#include "vec.cuh"

namespace linf {

struct NormDims {
    int N, C, G, L;             // samples, channels, groups, positions
    int Cg;                     // channels of a group
    double inv_m;               // 1 / (L * Cg)
};

// n / d of 0 <= n < 2^31 by a multiplication.
struct Divider {
    unsigned by, mul, shift;
    __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi((unsigned)n, mul) + (unsigned)n) >> shift); }
};
inline Divider make_divider(int by) {
    Divider d = {(unsigned)by, 0, 0};
    while ((1ull << d.shift) < (unsigned long long)by) ++d.shift;
    d.mul = (unsigned)(((1ull << 32) * ((1ull << d.shift) - (unsigned)by)) / (unsigned)by + 1);
    return d;
}

struct NormPlan {
    int V;                      // channels of a vector
    int groups;                 // groups of a column block (1 where a group is cut into pieces)
    int pieces, piece;          // column blocks of one group, vectors of such a block (pieces = 1: whole groups)
    int blocks;                 // column blocks
    int tx, rt;                 // threads along the channels and along the rows
    int same;                   // 1: all channels of a vector belong to one group
    int threads;                // of a CTA
    int kept;                   // 1: a CTA keeps a column block of a sample in shared memory, 0: two passes
    int splits, rows;           // CTAs that share a column block's rows (kept: 1), rows that a kept block has
    int per_cta, chunks;        // samples that a CTA takes one after the other (kept), CTAs along the samples
    Divider by_tx, by_blocks, by_cg;
};

// The column block of a CTA.
struct NormBlock { int c0, nvec, g0, ng, piece; };
template <int V>
__device__ __forceinline__ NormBlock norm_block(const NormDims& d, const NormPlan& p, int bx) {
    NormBlock b;
    if (p.pieces == 1) {
        b.g0 = bx * p.groups;
        b.ng = min(p.groups, d.G - b.g0);
        b.c0 = b.g0 * d.Cg;
        b.nvec = b.ng * d.Cg / V;
        b.piece = 0;
    } else {
        b.g0 = bx / p.pieces;
        b.ng = 1;
        b.piece = bx - b.g0 * p.pieces;
        b.c0 = b.g0 * d.Cg + b.piece * p.piece * V;
        b.nvec = min(p.piece, d.Cg / V - b.piece * p.piece);
    }
    return b;
}

// The groups (within the block) of channels c .. c + V - 1 of a block of whole groups; all 0 in a piece of a group.
template <int V>
__device__ __forceinline__ void groups_of(const NormDims& d, const NormPlan& p, int c, int (&g)[V]) {
    int at = 0, left = V;
    if (p.pieces == 1) {
        at = p.by_cg(c);
        left = (at + 1) * d.Cg - c;                               // channels of this group from c on
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (p.pieces == 1 && j > 0 && left == 0) { ++at; left = d.Cg; }
        --left;
        g[j] = at;
    }
}

// What a call reads: bytes of an element, tensors; whether it leaves per-channel sums behind (then a CTA takes several small samples).
struct NormKind { int elem_bytes, tensors; bool sums; };

constexpr int kNormThreads = 256;
constexpr int kNormKeepBytes = 64 * 1024; // of a CTA, so that an SM has three
constexpr int kNormSplits = 64;           // CTAs that share a block's rows in the two passes: one of the second adds up that many sums
constexpr int kNormSamples = 32;          // samples whose sums a kept CTA adds up in fp32 at most
constexpr int kNormPlaces = 4;            // CTAs of the two passes that an SM has at a time, about

inline int norm_ceil(long long a, long long b) { return (int)((a + b - 1) / b); }

// widest vector of {16, 8, 4 bytes, one element} that the call allows, and the least number of groups whose channels make whole
// vectors; `cap`: vectors along the channels of a CTA.  One group may be wider than `cap`: *kmin = 0 then (it has to be cut).
inline int norm_vector(const NormDims& d, int elem_bytes, bool aligned, int cap, int* kmin) {
    const int widths[4] = {16 / elem_bytes, 8 / elem_bytes, 4 / elem_bytes, 1};
    for (int k = 0; k < 4; ++k) {
        const int V = widths[k];
        if (V > 1 && (!aligned || d.C % V != 0)) continue;
        int a = d.Cg, b = V;
        while (b != 0) { const int r = a % b; a = b; b = r; }
        *kmin = V / a;                                            // divides G, for V divides G * Cg
        if ((long long)*kmin * d.Cg / V <= cap) return V;
        if (*kmin == 1) { *kmin = 0; return V; }                  // else narrower vectors divide the group
    }
    return 1;                                                     // not reached: V = 1 has kmin = 1
}

inline void norm_columns(const NormDims& d, NormPlan* p, int kmin, int units) {
    const int all = d.G / kmin;
    int blocks = norm_ceil(all, units);
    const int each = norm_ceil(all, blocks);
    p->blocks = norm_ceil(all, each);
    p->groups = each * kmin;
    p->pieces = 1;
    p->piece = 0;
    p->tx = (int)((long long)p->groups * d.Cg / p->V);
}

inline bool norm_keep(const NormDims& d, const NormKind& kind, bool aligned, NormPlan* p) {
    int kmin;
    p->V = norm_vector(d, kind.elem_bytes, aligned, kNormThreads, &kmin);
    if (kmin == 0) return false;
    const long long unit = (long long)kmin * d.Cg / p->V;                   // vectors of the narrowest column block
    const long long row_bytes = unit * p->V * kind.elem_bytes;
    auto bytes = [&](long long units) { return units * row_bytes * kind.tensors * d.L; };
    if (bytes(1) > kNormKeepBytes) return false;
    // Wider blocks while a row's piece is under 64 bytes (two sectors of L2), or while there are CTAs enough for the whole GPU several times
    // over with few bytes each
    int units = 1;
    while (units * kmin < d.G && 2 * units * unit <= kNormThreads && bytes(2 * units) <= kNormKeepBytes) {
        const long long ctas = (long long)d.N * norm_ceil(d.G / kmin, units);
        const bool narrow = units * row_bytes < 64, many = ctas > 8LL * sm_count() && bytes(2 * units) <= 16 * 1024;
        if (!narrow && !many) break;
        units *= 2;
    }
    if (units * row_bytes < 32 && units * kmin < d.G && d.L > 1) return false;      // half a sector: two passes over whole rows are faster
    norm_columns(d, p, kmin, units);
    p->rows = d.L;
    p->splits = 1;
    // about four vectors to a thread where there are few, 256 threads otherwise
    long long threads = (long long)p->tx * norm_ceil(p->rows, 4);
    if (threads < 64) threads = 64;
    if (threads > kNormThreads) threads = kNormThreads;
    if (threads < p->tx) threads = p->tx;
    p->rt = (int)(threads / p->tx);
    if (p->rt > p->rows) p->rt = p->rows;
    p->threads = norm_ceil((long long)p->tx * p->rt, 32) * 32;
    p->kept = 1;
    // with per-channel sums: as many CTAs as run at a time, twice over; a CTA adds its samples up in order
    const long long resident = (long long)sm_count() * (2048 / p->threads < 16 ? 2048 / p->threads : 16) * 2;
    p->per_cta = kind.sums ? norm_ceil((long long)d.N * p->blocks, resident) : 1;
    if (p->per_cta > kNormSamples) p->per_cta = kNormSamples;
    p->chunks = norm_ceil(d.N, p->per_cta);
    return true;
}

inline void norm_two_passes(const NormDims& d, const NormKind& kind, bool aligned, NormPlan* p) {
    int kmin;
    const int cap = kNormThreads;
    p->V = norm_vector(d, kind.elem_bytes, aligned, cap, &kmin);
    if (kmin == 0) {
        p->groups = 1;
        const int vecs = d.Cg / p->V;
        p->pieces = norm_ceil(vecs, cap);
        p->piece = norm_ceil(vecs, p->pieces);
        p->pieces = norm_ceil(vecs, p->piece);
        p->blocks = d.G * p->pieces;
        p->tx = p->piece;
    } else {
        norm_columns(d, p, kmin, (int)(cap / ((long long)kmin * d.Cg / p->V)));
    }
    p->threads = kNormThreads;
    p->rt = cap / p->tx;
    if (p->rt > d.L) p->rt = d.L;
    // as few CTAs to a block as fill the GPU's places nearly whole (one CTA more than fits costs a wave: 31 instead of 26 us for the sums of
    // 32 x 320 x 64 x 64 bf16), with at least four rows for each thread
    const long long ctas = (long long)p->blocks * d.N, places = (long long)sm_count() * kNormPlaces;
    long long most = norm_ceil(d.L, 4LL * p->rt), s = 1;
    if (most > kNormSplits) most = kNormSplits;
    double best = 0.0;
    for (long long k = 1; k <= most && best < 0.9; ++k) {
        const double full = (double)(ctas * k) / (double)(norm_ceil(ctas * k, places) * places);
        if (full > best) { best = full; s = k; }
    }
    p->rows = 0;
    p->splits = (int)s;                                         // splits * rt <= L: every thread has a row
    p->per_cta = 1;
    p->chunks = d.N;
}

// A call's dimensions and plan: LINF_OK or the refusal.
inline int norm_make(int N, int C, int G, int L, const NormKind& kind, bool aligned, NormDims* d, NormPlan* p) {
    if (N <= 0 || C <= 0 || G <= 0 || L <= 0) return LINF_ERR_DIMS;
    if (C % G != 0) return LINF_ERR_GROUP;
    if (N > (1 << 30) || L > (1 << 30)) return LINF_ERR_TOO_LARGE;
    d->N = N; d->C = C; d->G = G; d->L = L; d->Cg = C / G;
    d->inv_m = 1.0 / ((double)L * d->Cg);
    *p = NormPlan{};
    if (!norm_keep(*d, kind, aligned, p)) {
        *p = NormPlan{};
        norm_two_passes(*d, kind, aligned, p);
    }
    p->same = d->Cg % p->V == 0;
    p->by_tx = make_divider(p->tx);
    p->by_blocks = make_divider(p->blocks);
    p->by_cg = make_divider(d->Cg);
    if ((long long)N * p->blocks * p->splits > 0x7fffffffLL) return LINF_ERR_TOO_LARGE;
    return LINF_OK;
}

// One position (group_norm_dense.cu): a row of C/G values belongs to a slot of `tpr` threads; a CTA has slots for `groups` groups times `subs`
// samples, and takes `per` samples.
constexpr int kDenseSamples = 64;
struct DensePlan { int V, tpr, threads, groups, subs, blocks, per, chunks; };
struct NormGiven;
bool dense_plan(const NormDims& d, int elem_bytes, bool aligned, int ctas, DensePlan* p);
int dense_norm_forward(const void* x, const NormGiven& given, const NormDims& d, const DensePlan& p, int type, double eps, int act, const Drop& drop,
                       void* y, float* mean, float* rstd, cudaStream_t st);
// by_channel: chunks * subs rows of C
int dense_norm_backward(const void* dy, const void* x, const NormGiven& given, const float* mean, const float* rstd, const NormDims& d, const DensePlan& p,
                        int type, int act, const Drop& drop, void* dx, float2* by_channel, cudaStream_t st);

// dgamma and dbeta from `count` rows of per-channel sums (du, du h); either may be null (group_norm.cu).  A CTA has 8 channels.
inline unsigned norm_param_ctas(int C) { return (unsigned)norm_ceil(C, 8); }
int norm_params(const float2* by_channel, long long count, int C, void* dgamma, void* dbeta, int ptype, cudaStream_t st);

// gamma and beta, or what stands for them where they are null, and a generator state that stands for one that is not needed, on the
// current device; false if CUDA refused (group_norm.cu)
struct NormGiven { Param gamma, beta; const long long* idle; };
bool norm_given(const void* gamma, const void* beta, int ptype, NormGiven* g);

template <typename X> __device__ __forceinline__ X* space_at(uint4* space, size_t at) { return reinterpret_cast<X*>(reinterpret_cast<char*>(space) + at); }

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The rows of a CTA: the threads of all row ranges take the sample's rows in turn, so that CTAs that run side by side read side by side.  A thread
// has `base` rows, or one more in the first `more` of the CTA's rows of threads.
struct NormRows { int base, more, all; };
__device__ __forceinline__ NormRows norm_rows(const NormDims& d, const NormPlan& p, int split) {
    const int threads = p.splits * p.rt;
    NormRows r;
    r.base = d.L / threads;
    r.more = min(max(d.L - r.base * threads - split * p.rt, 0), p.rt);
    r.all = r.base * p.rt + r.more;
    return r;
}
__device__ __forceinline__ int rows_of(const NormRows& r, int rt) { return r.base + (rt < r.more ? 1 : 0); }

// Columns c of [0, width), each with as many neighbouring lanes as the CTA has to spare, up to a warp: body(c, first row, step, join) adds the
// rows first, first + step, ... up and calls join(s, t), which adds both over the lanes and is true in the one that keeps them.  c >= width
// comes with no rows.
template <typename Body>
__device__ __forceinline__ void by_columns(int width, int rows, Body body) {
    int lanes = 1;
    while (lanes < 32 && 2 * lanes * width <= (int)blockDim.x && lanes < rows) lanes *= 2;
    const int at_a_time = blockDim.x / lanes, mine = threadIdx.x / lanes, part = threadIdx.x - mine * lanes;
    for (int c0 = 0; c0 < width; c0 += at_a_time) {
        const int c = c0 + mine;
        body(c, c < width ? part : rows, lanes, [&](auto& s, auto& t) {
            for (int o = 1; o < lanes; o *= 2) {
                s += __shfl_xor_sync(0xffffffffu, s, o);
                t += __shfl_xor_sync(0xffffffffu, t, o);
            }
            return c < width && part == 0;
        });
    }
}

template <int BYTES>
__device__ __forceinline__ void copy_shared(unsigned to, const void* from) {
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else if (BYTES == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
// One vector of a kept row from global to shared memory, asynchronously where its size allows.
template <typename T, int V>
__device__ __forceinline__ void keep_vector(T* to, const T* from) {
    constexpr int bytes = sizeof(T) * V;
    if constexpr (bytes >= 4) copy_shared<bytes>((unsigned)__cvta_generic_to_shared(to), from);
    else *to = *from;
}
__device__ __forceinline__ void keep_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }      // a thread reads only what it copied itself

template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_shared(unsigned at) {
    Raw<T, V> v;
    if constexpr (sizeof(T) * V == 16) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    else if constexpr (sizeof(T) * V == 8) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(*reinterpret_cast<unsigned*>(&v)) : "r"(at) : "memory");
    return v;
}

template <typename T, int V, int N, int S>
__host__ __device__ constexpr size_t norm_ring_bytes() { return sizeof(T) * V >= 4 ? (size_t)kNormThreads * sizeof(T) * V * N * S : 0; }

// The rows first, first + every, ... below `end` of a thread's column in each of N tensors (at[k] points at row 0).  S rows are on their way
// to shared memory at a time, each thread's to places of its own (`ring`: norm_ring_bytes), so that neither registers nor barriers limit
// how much is read ahead (32 x 320 x 64 x 64 bf16, both passes: batches of 8 loads to registers 68 us, this 59 us).  Elements of two bytes that no wider copy
// reaches come through registers.
template <typename T, int V, int N, int S>
struct NormStream {
    static constexpr int bytes = sizeof(T) * V, place = kNormThreads * bytes;      // ring: [S][N][threads]
    unsigned own;
    const T* next[N];
    size_t stride;
    int r, r1, step, ahead;

    // starts with the first rows on their way: what the CTA does before run(rows, body(row, vectors)) overlaps with them
    __device__ __forceinline__ NormStream(void* ring, const T* const (&at)[N], int first, int end, int every, size_t C) {
        r = ahead = first;
        r1 = end;
        step = every;
        stride = (size_t)every * C;
#pragma unroll
        for (int k = 0; k < N; ++k) next[k] = at[k] + (size_t)first * C;
        if constexpr (bytes >= 4) {
            own = (unsigned)__cvta_generic_to_shared(ring) + threadIdx.x * bytes;
#pragma unroll
            for (int s = 0; s < S; ++s) issue(s);
        }
    }
    __device__ __forceinline__ void issue(int s) {
        if (ahead < r1) {
#pragma unroll
            for (int k = 0; k < N; ++k) {
                copy_shared<bytes>(own + (s * N + k) * place, next[k]);
                next[k] += stride;
            }
        }
        ahead += step;
        cp_async_commit();
    }
    template <typename Body> __device__ __forceinline__ void row(int s, Body& body) {
        cp_async_wait<S - 1>();
        Raw<T, V> v[N];
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = load_shared<T, V>(own + (s * N + k) * place);
        body(r, v);
        issue(s);                                               // behind body, which has used what it overwrites
        r += step;
    }
    // The next `rows` rows of the thread, a multiple of S but for the last ones.
    // LIGHT bodies are written out for a whole turn of the ring: half the instructions (sums of bf16 maps: 52 -> 34 a vector, 24 -> 21 us);
    // heavy ones are not, their code would be too long (38 -> 40 us).
    template <bool LIGHT, typename Body> __device__ __forceinline__ void run(int rows, Body body) {
        const int end = r + rows * step;                        // below L + step
        if constexpr (LIGHT && bytes >= 4) {
            for (int turns = rows / S; turns > 0; --turns) {
#pragma unroll
                for (int s = 0; s < S; ++s) row(s, body);
            }
        }
        run_to(end, body);
    }
    template <typename Body> __device__ __forceinline__ void run_all(Body body) { run_to(r1, body); }
    template <typename Body> __device__ __forceinline__ void run_to(int end, Body& body) {
        if constexpr (bytes >= 4) {
#pragma unroll 1
            for (int s = 0; r < end; s = s + 1 == S ? 0 : s + 1) row(s, body);
        } else {
            constexpr int K = S;
            for (; r < end; r += K * step) {
                Raw<T, V> v[K][N];
#pragma unroll
                for (int j = 0; j < K; ++j) {
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        if (r + j * step < end) v[j][k] = load_raw<T, V>(next[k]);
                        next[k] += stride;
                    }
                }
#pragma unroll
                for (int j = 0; j < K; ++j)
                    if (r + j * step < end) body(r + j * step, v[j]);
            }
        }
    }
};

// Lets a kernel have more than 48 KB of dynamic shared memory, once for each device and to the device's limit: the limit is the kernel's on that
// device, not the call's, and one that followed each call's size would fall under that of another host thread's launch.
template <auto kernel>
bool allow_shared(size_t bytes) {
    static std::atomic<bool> known[kMaxDevices];
    if (bytes <= 48 * 1024) return true;
    int dev = -1, most = 0;
    if (cudaGetDevice(&dev) == cudaSuccess) {
        if (dev < kMaxDevices && known[dev].load(std::memory_order_relaxed)) return true;
        if (cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev) == cudaSuccess &&
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most) == cudaSuccess) {
            if (dev < kMaxDevices) known[dev].store(true, std::memory_order_relaxed);
            return true;
        }
    }
    cudaGetLastError();
    return false;
}

// ---- launches that begin before the kernel in front has ended ---------------------------------------------------------
// The kernel in front lets the next one's CTAs in where its own have left (all of its CTAs are running by then); what it wrote is read
// behind grid_wait(), which returns when it has ended, and with loads that go to L2 (__ldcg), which nothing moves in front of it.  What the
// CTAs do before that overlaps with its end and with the launch itself (2 to 4 us of a pair).
__device__ __forceinline__ void grid_let_go() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... A, typename... B>
int launch_behind(void (*kernel)(A...), dim3 grid, int threads, size_t shared, cudaStream_t st, B... args) {
    cudaLaunchConfig_t c = {};
    c.gridDim = grid;
    c.blockDim = dim3((unsigned)threads);
    c.dynamicSmemBytes = shared;
    c.stream = st;
    cudaLaunchAttribute a = {};
    a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &a;
    c.numAttrs = 1;
    if (cudaLaunchKernelEx(&c, kernel, A(args)...) != cudaSuccess) {
        cudaGetLastError();
        return LINF_ERR_LAUNCH;
    }
    return launch_status();
}

// A kept call.
template <auto kernel, typename... B>
int launch_kept(const NormPlan& p, size_t shared, cudaStream_t st, B... args) {
    if (!allow_shared<kernel>(shared)) return LINF_ERR_LAUNCH;
    kernel<<<(unsigned)(p.chunks * p.blocks), p.threads, shared, st>>>(args...);
    return launch_status();
}

}  // namespace linf
