// Element types, wide loads and the maps that the operators between two layers share (group norm, dropout).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace linf {

// ---- V neighbouring elements of type T as one load / store --------------------------------------------------
template <int BYTES> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = unsigned; };
template <> struct RawOf<2> { using type = unsigned short; };

template <typename T, int V> using Raw = typename RawOf<(int)sizeof(T) * V>::type;

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
// one rounding to nearest at the end of each 16-bit output; everything before it is fp32
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int V>
__device__ __forceinline__ void unpack(const Raw<T, V>& raw, float (&f)[V]) {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = to_float<T>(e[j]);
}
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> pack(const float (&f)[V]) {
    Raw<T, V> raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int j = 0; j < V; ++j) e[j] = from_float<T>(f[j]);
    return raw;
}
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p) { return *reinterpret_cast<const Raw<T, V>*>(p); }
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_once(const T* p) { return __ldcs(reinterpret_cast<const Raw<T, V>*>(p)); }
template <typename T, int V>
__device__ __forceinline__ void store_once(T* p, const Raw<T, V>& v) { __stcs(reinterpret_cast<Raw<T, V>*>(p), v); }

// a parameter vector of float or of the activations' 16-bit type
__device__ __forceinline__ float load_param(const void* p, int c, int type) {
    if (type == LINF_F32) return __ldg(static_cast<const float*>(p) + c);
    if (type == LINF_F16) return __half2float(__ldg(static_cast<const __half*>(p) + c));
    return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p) + c));
}
__device__ __forceinline__ void store_param(void* p, int c, int type, float v) {
    if (type == LINF_F32) static_cast<float*>(p)[c] = v;
    else if (type == LINF_F16) static_cast<__half*>(p)[c] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[c] = __float2bfloat16_rn(v);
}

// ---- activations: the value, and the value's derivative ---------------------------------------------------------
// silu(u) = u / (1 + e^-u) has one minimum, at u = kSiluArg; it falls before and rises behind it
constexpr double kSiluArg64 = -1.278464542761074;
constexpr float kSiluArg = (float)kSiluArg64;

__device__ __forceinline__ float sigmoid(float u) { return __fdividef(1.f, 1.f + __expf(-u)); }   // both ends come out as 1 and 0
__device__ __forceinline__ float activate(float u, int act) {
    switch (act) {
        case LINF_ACT_RELU: return u < 0.f ? 0.f : u;            // keeps a NaN
        case LINF_ACT_TANH: return tanhf(u);
        case LINF_ACT_SILU: return u * sigmoid(u);
        default: return u;
    }
}
__device__ __forceinline__ float slope(float u, int act) {
    switch (act) {
        case LINF_ACT_RELU: return u > 0.f ? 1.f : 0.f;
        case LINF_ACT_TANH: { const float t = tanhf(u); return 1.f - t * t; }
        case LINF_ACT_SILU: { const float q = sigmoid(u); return q * (1.f + u * (1.f - q)); }
        default: return 1.f;
    }
}

// ---- counter-based dropout --------------------------------------------------------------------------------------
// Philox4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011; 7 is the least
// number of rounds for which they report no failure of the BigCrush battery).  Element i of a tensor takes 16 bits, piece i % 8 of the four
// words that the counter (i / 8, offset) gives under the key `seed`, and is kept where that piece is at least
// threshold = round(rate * 2^16).  So a mask is a function of (seed, offset, i) alone and is computed again by the backward pass
// instead of being stored.  Sixteen bits and not 32: rates then count in steps of 2^-16, and the scale 2^16 / (2^16 - threshold)
// makes up for the rounded rate, so that the expectation is exact.  With 32 bits and 10 rounds a pass over 64 Mi bf16 values took 72 us
// for the integer multiplications alone, with 16 bits 49 us, without a generator 44 us.
struct Drop {
    const long long* rng;       // {seed, offset} on the device, null = no dropout
    unsigned threshold;         // 0 .. 65536
    float scale;
};
struct DropKey { unsigned k0, k1, o0, o1; };

__device__ __forceinline__ DropKey drop_key(const Drop& d) {
    const unsigned long long seed = (unsigned long long)__ldg(d.rng), off = (unsigned long long)__ldg(d.rng + 1);
    return DropKey{(unsigned)seed, (unsigned)(seed >> 32), (unsigned)off, (unsigned)(off >> 32)};
}
__device__ __forceinline__ uint4 drop_words(const DropKey& k, unsigned long long block) {
    uint4 c = make_uint4((unsigned)block, (unsigned)(block >> 32), k.o0, k.o1);
    unsigned k0 = k.k0, k1 = k.k1;
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const unsigned long long a = (unsigned long long)0xD2511F53u * c.x, b = (unsigned long long)0xCD9E8D57u * c.z;
        c = make_uint4((unsigned)(b >> 32) ^ c.y ^ k0, (unsigned)b, (unsigned)(a >> 32) ^ c.w ^ k1, (unsigned)a);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return c;
}
// f[j] of element i0 + j (i0 a multiple of V): scaled where it is kept, 0 where not (whatever the value was, a NaN included)
template <int V>
__device__ __forceinline__ void drop_apply(const Drop& d, const DropKey& k, unsigned long long i0, float (&f)[V]) {
    const uint4 w = drop_words(k, i0 >> 3);
    if (V == 8) {
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const unsigned piece = (j & 1) ? u[(j >> 1) & 3] >> 16 : u[(j >> 1) & 3] & 0xffffu;
            f[j] = piece >= d.threshold ? f[j] * d.scale : 0.f;
        }
    } else {
        // the 64 bits that hold the pieces of this element's half of the block, shifted to its first piece
        const bool second = (i0 & 4) != 0;
        unsigned long long bits = second ? ((unsigned long long)w.w << 32 | w.z) : ((unsigned long long)w.y << 32 | w.x);
        if (V < 4) bits >>= 16 * (unsigned)(i0 & 3);
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = (unsigned)((bits >> (16 * (j & 3))) & 0xffffu) >= d.threshold ? f[j] * d.scale : 0.f;
    }
}

// threshold and scale of a rate in [0, 1]; false outside (a NaN included).  Rate 1 keeps nothing.
inline bool make_drop(double rate, const long long* rng, Drop* d) {
    if (!(rate >= 0.0 && rate <= 1.0)) return false;
    d->threshold = (unsigned)(rate * 65536.0 + 0.5);
    d->scale = d->threshold < 65536u ? (float)(65536.0 / (65536.0 - (double)d->threshold)) : 0.f;
    d->rng = d->threshold > 0 ? rng : nullptr;      // a threshold of 0 keeps every element as it is
    return true;
}

}  // namespace linf
