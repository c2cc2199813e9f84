// How the group-norm kernels deal a [N, L, C] activation (channels last) out to CTAs.
//
// A CTA takes a column block -- some whole groups, or a piece of one group -- and a range of rows (positions) of one sample.
// Its threads form RT rows of TX vectors; a thread keeps its column, so that parameters and per-channel sums stay in registers.
// Vectors are as wide as C, the groups and the pointers' alignment allow: a block of whole groups starts and ends on a vector.
#pragma once

#include "vec.cuh"

namespace linf {

constexpr int kNormThreads = 256;
constexpr int kNormMaxGroups = 2048;      // groups of one column block: 256 vectors of at most 8 channels

struct NormDims {
    int N, C, G, L;             // samples, channels, groups, positions
    int Cg;                     // channels of a group
    double inv_m;               // 1 / (L * Cg)
};

struct NormPlan {
    int V;                      // channels of a vector
    int groups;                 // groups of a column block (1 where a group is cut into pieces)
    int pieces, piece;          // column blocks of one group, vectors of such a block (pieces = 1: whole groups)
    int blocks;                 // column blocks
    int tx, rt;                 // threads along the channels and along the rows
    int splits, rows;           // row ranges of a sample, rows of a range
};

// The column block of a CTA.
struct NormBlock { int c0, nvec, g0, ng, piece; };
__device__ __forceinline__ NormBlock norm_block(const NormDims& d, const NormPlan& p, int bx) {
    NormBlock b;
    if (p.pieces == 1) {
        b.g0 = bx * p.groups;
        b.ng = min(p.groups, d.G - b.g0);
        b.c0 = b.g0 * d.Cg;
        b.nvec = b.ng * d.Cg / p.V;
        b.piece = 0;
    } else {
        b.g0 = bx / p.pieces;
        b.ng = 1;
        b.piece = bx - b.g0 * p.pieces;
        b.c0 = b.g0 * d.Cg + b.piece * p.piece * p.V;
        b.nvec = min(p.piece, d.Cg / p.V - b.piece * p.piece);
    }
    return b;
}

// The largest vector of {16 bytes, 4 bytes, one element} that the call allows; cap = vectors along the channels of a CTA.
inline NormPlan norm_plan(const NormDims& d, int elem_bytes, bool aligned, int cap) {
    NormPlan p = {};
    const int widths[3] = {16 / elem_bytes, 4 / elem_bytes, 1};
    for (int k = 0; k < 3; ++k) {
        const int V = widths[k];
        if (k > 0 && V == widths[k - 1]) continue;
        if (V > 1 && (!aligned || d.C % V != 0)) continue;
        int a = d.Cg, b = V;
        while (b != 0) { const int r = a % b; a = b; b = r; }
        const int kmin = V / a;                                   // groups whose channels make whole vectors
        const long long need = (long long)kmin * d.Cg / V;
        if (need > cap) {
            if (kmin != 1) continue;                              // narrower vectors divide the group
            p.V = V;
            p.groups = 1;
            const int vecs = d.Cg / V;
            p.pieces = (vecs + cap - 1) / cap;
            p.piece = (vecs + p.pieces - 1) / p.pieces;
            p.pieces = (vecs + p.piece - 1) / p.piece;
            p.blocks = d.G * p.pieces;
            p.tx = p.piece;
        } else {
            p.V = V;
            const int units = d.G / kmin;                         // kmin divides G, for V divides G * Cg
            const int per = (int)(cap / need);
            int blocks = (units + per - 1) / per;
            const int each = (units + blocks - 1) / blocks;
            blocks = (units + each - 1) / each;
            p.groups = each * kmin;
            p.pieces = 1;
            p.piece = 0;
            p.blocks = blocks;
            p.tx = p.groups * d.Cg / V;
        }
        break;
    }
    p.rt = cap / p.tx;
    return p;
}

// Row ranges: enough CTAs for the GPU, at least four rows for each thread, at most `most` ranges (whoever adds them up reads that many).
inline void norm_split_rows(const NormDims& d, NormPlan* p, int most) {
    const long long ctas = (long long)p->blocks * d.N, want = (long long)sm_count() * 8;
    long long s = ctas >= want ? 1 : (want + ctas - 1) / ctas;
    const long long by_rows = (d.L + 4LL * p->rt - 1) / (4LL * p->rt);
    if (s > by_rows) s = by_rows;
    if (s > most) s = most;
    if (s < 1) s = 1;
    p->rows = (int)((d.L + s - 1) / s);
    p->splits = (d.L + p->rows - 1) / p->rows;
}

// A call's dimensions and plan: LINF_OK or the refusal.
constexpr int kNormSplits = 64;           // row ranges of a sample at most

inline int norm_make(int N, int C, int G, int L, int elem_bytes, bool aligned, NormDims* d, NormPlan* p) {
    if (N <= 0 || C <= 0 || G <= 0 || L <= 0) return LINF_ERR_DIMS;
    if (C % G != 0) return LINF_ERR_GROUP;
    d->N = N; d->C = C; d->G = G; d->L = L; d->Cg = C / G;
    d->inv_m = 1.0 / ((double)L * d->Cg);
    *p = norm_plan(*d, elem_bytes, aligned, kNormThreads);
    if (L > (1 << 30) || (long long)N * p->blocks > 0x7fffffffLL) return LINF_ERR_TOO_LARGE;
    norm_split_rows(*d, p, kNormSplits);
    return LINF_OK;
}

// dgamma and dbeta from `count` rows of per-channel sums (du, du h); either may be null (group_norm.cu)
int norm_params(const float2* by_channel, long long count, int C, void* dgamma, void* dbeta, int ptype, cudaStream_t st);

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

}  // namespace linf
