// Element types, wide loads and the maps that the operators between two layers share (group norm, dropout).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

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
    const unsigned* w = reinterpret_cast<const unsigned*>(&raw);
    if (sizeof(T) == 2 && V > 1) {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {                           // two elements of a word: one operation each
            if (std::is_same<T, __nv_bfloat16>::value) {
                f[2 * j] = __uint_as_float(w[j] << 16);
                f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            } else {
                const float2 p = __half22float2(*reinterpret_cast<const __half2*>(w + j));
                f[2 * j] = p.x;
                f[2 * j + 1] = p.y;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = to_float<T>(e[j]);
    }
}
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> pack(const float (&f)[V]) {
    Raw<T, V> raw;
    T* e = reinterpret_cast<T*>(&raw);
    if (sizeof(T) == 2 && V > 1) {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            if (std::is_same<T, __nv_bfloat16>::value) reinterpret_cast<__nv_bfloat162*>(&raw)[j] = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
            else reinterpret_cast<__half2*>(&raw)[j] = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) e[j] = from_float<T>(f[j]);
    }
    return raw;
}
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p) { return *reinterpret_cast<const Raw<T, V>*>(p); }
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_once(const T* p) { return __ldcs(reinterpret_cast<const Raw<T, V>*>(p)); }
template <typename T, int V>
__device__ __forceinline__ void store_once(T* p, const Raw<T, V>& v) { __stcs(reinterpret_cast<Raw<T, V>*>(p), v); }

// A parameter vector, fp32 or of the activations' 16-bit type; kind PARAM_ONE: one value in the place of a vector that was not given, so
// that no kernel holds a pointer that it must not follow; PARAM_WIDE: fp32 on a 16-byte boundary.
enum { PARAM_ONE, PARAM_WIDE, PARAM_F32, PARAM_F16, PARAM_BF16 };
struct Param { const void* at; int kind; };
__device__ __forceinline__ float load_param(const Param& p, int c) {
    if (p.kind == PARAM_ONE) return __ldg(static_cast<const float*>(p.at));
    if (p.kind <= PARAM_F32) return __ldg(static_cast<const float*>(p.at) + c);
    if (p.kind == PARAM_F16) return __half2float(__ldg(static_cast<const __half*>(p.at) + c));
    return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p.at) + c));
}
// the values of channels c .. c + V - 1 (c a multiple of V)
template <int V>
__device__ __forceinline__ void load_params(const Param& p, int c, float (&f)[V]) {
    if (V % 4 == 0 && p.kind == PARAM_WIDE) {
#pragma unroll
        for (int j = 0; j < V / 4; ++j) {
            const float4 q = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.at) + c) + j);
            f[4 * j] = q.x;
            f[4 * j + 1] = q.y;
            f[4 * j + 2] = q.z;
            f[4 * j + 3] = q.w;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = load_param(p, c + j);
}
__device__ __forceinline__ void store_param(void* p, int c, int type, float v) {
    if (type == LINF_F32) static_cast<float*>(p)[c] = v;
    else if (type == LINF_F16) static_cast<__half*>(p)[c] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[c] = __float2bfloat16_rn(v);
}

// ---- V fp32 values at a time, two to a register pair and an instruction ------------------------------------------
template <int V> struct Lanes {
    unsigned long long p[V / 2];
    __device__ __forceinline__ void get(float (&f)[V]) const {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) unpack_f32x2(p[j], f[2 * j], f[2 * j + 1]);
    }
    __device__ __forceinline__ void set(const float (&f)[V]) {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) p[j] = pack_f32x2(f[2 * j], f[2 * j + 1]);
    }
    __device__ __forceinline__ void fill(float f) {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) p[j] = pack_f32x2(f, f);
    }
};
template <> struct Lanes<1> {
    float p[1];
    __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = p[0]; }
    __device__ __forceinline__ void set(const float (&f)[1]) { p[0] = f[0]; }
    __device__ __forceinline__ void fill(float f) { p[0] = f; }
};
#define LINF_LANES(name, scalar, packed)                                                                   \
    template <int V> __device__ __forceinline__ Lanes<V> name(const Lanes<V>& a, const Lanes<V>& b) {      \
        Lanes<V> r;                                                                                        \
        _Pragma("unroll") for (int j = 0; j < V / 2; ++j) r.p[j] = packed(a.p[j], b.p[j]);                 \
        return r;                                                                                          \
    }                                                                                                      \
    __device__ __forceinline__ Lanes<1> name(const Lanes<1>& a, const Lanes<1>& b) {                       \
        Lanes<1> r;                                                                                        \
        r.p[0] = a.p[0] scalar b.p[0];                                                                     \
        return r;                                                                                          \
    }
// (no difference: the packed addition takes no sign, and turning the signs of a pair costs two operations)
LINF_LANES(add, +, add_f32x2)
LINF_LANES(mul, *, mul_f32x2)
#undef LINF_LANES
template <int V> __device__ __forceinline__ Lanes<V> fma(const Lanes<V>& a, const Lanes<V>& b, const Lanes<V>& c) {
    Lanes<V> r;
#pragma unroll
    for (int j = 0; j < V / 2; ++j) r.p[j] = fma_f32x2(a.p[j], b.p[j], c.p[j]);
    return r;
}
__device__ __forceinline__ Lanes<1> fma(const Lanes<1>& a, const Lanes<1>& b, const Lanes<1>& c) {
    Lanes<1> r;
    r.p[0] = fmaf(a.p[0], b.p[0], c.p[0]);
    return r;
}
template <int V> __device__ __forceinline__ Lanes<V> filled(float f) { Lanes<V> r; r.fill(f); return r; }
template <int V> __device__ __forceinline__ Lanes<V> lanes(const float (&f)[V]) { Lanes<V> r; r.set(f); return r; }
template <typename T, int V>
__device__ __forceinline__ Lanes<V> lanes_of(const Raw<T, V>& raw) {
    float f[V];
    unpack<T, V>(raw, f);
    return lanes<V>(f);
}
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> raw_of(const Lanes<V>& v) {
    float f[V];
    v.get(f);
    return pack<T, V>(f);
}
template <typename T, int V> __device__ __forceinline__ Lanes<V> load_lanes(const T* p) { return lanes_of<T, V>(load_raw<T, V>(p)); }

// ---- activations: the value, and the value's derivative ---------------------------------------------------------
// silu(u) = u / (1 + e^-u) has one minimum, at u = kSiluArg; it falls before and rises behind it
constexpr double kSiluArg64 = -1.278464542761074;
constexpr float kSiluArg = (float)kSiluArg64;

// 2^x and 1 / x of the special-function unit (relative error 2^-22 and 2^-23 by their specification; subnormals count as 0)
__device__ __forceinline__ float exp2_unit(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float rcp_unit(float x) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
constexpr float kLog2E = 1.44269504088896f;

// tanh for results that are rounded to 16 bits: 1 - 2 / (1 + e^2u) is off by up to 2^-22, which is below a half step of the
// result's type from |u| = 2^-4 on; below, the series to u^5 is off by 17/315 u^7, less than 2^-28 of u
__device__ __forceinline__ float tanh16(float u) {
    const float s = u * u, series = u * fmaf(s, fmaf(s, 2.f / 15.f, -1.f / 3.f), 1.f);
    const float far = fmaf(-2.f, rcp_unit(1.f + exp2_unit(2.f * kLog2E * u)), 1.f);
    return s < 1.f / 256.f ? series : far;
}
template <bool WIDE> __device__ __forceinline__ float tanh_of(float u) { return WIDE ? tanhf(u) : tanh16(u); }

// 1 / (1 + e^-u): both ends come out as 1 and 0
template <int V> __device__ __forceinline__ Lanes<V> sigmoid(const Lanes<V>& u) {
    float f[V];
    mul(u, filled<V>(-kLog2E)).get(f);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = exp2_unit(f[j]);
    add(lanes<V>(f), filled<V>(1.f)).get(f);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = rcp_unit(f[j]);
    return lanes<V>(f);
}

// WIDE: the results stay fp32.
template <bool WIDE, int V>
__device__ __forceinline__ Lanes<V> activate(const Lanes<V>& u, int act) {
    if (act == LINF_ACT_IDENTITY) return u;
    if (act == LINF_ACT_SILU) return mul(u, sigmoid<V>(u));
    float f[V];
    u.get(f);
    if (act == LINF_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = f[j] < 0.f ? 0.f : f[j];          // keeps a NaN
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = tanh_of<WIDE>(f[j]);
    }
    return lanes<V>(f);
}
template <bool WIDE, int V>
__device__ __forceinline__ Lanes<V> slope(const Lanes<V>& u, int act) {
    const Lanes<V> one = filled<V>(1.f);
    if (act == LINF_ACT_IDENTITY) return one;
    if (act == LINF_ACT_SILU) {
        const Lanes<V> q = sigmoid<V>(u);
        return mul(fma(u, fma(q, filled<V>(-1.f), one), one), q);
    }
    float f[V];
    u.get(f);
    if (act == LINF_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = f[j] > 0.f ? 1.f : 0.f;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) { const float t = tanh_of<WIDE>(f[j]); f[j] = fmaf(-t, t, 1.f); }
    }
    return lanes<V>(f);
}
__device__ __forceinline__ float activate(float u, int act) { return activate<true, 1>(filled<1>(u), act).p[0]; }
__device__ __forceinline__ float slope(float u, int act) { return slope<true, 1>(filled<1>(u), act).p[0]; }

// ---- counter-based dropout --------------------------------------------------------------------------------------
// Philox4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011; 7 is the least
// number of rounds for which they report no failure of the BigCrush battery).  Element i of a tensor takes 16 bits, piece i % 8 of the four
// words that the counter (i / 8, offset) gives under the key `seed`, and is kept where that piece is at least
// threshold = round(rate * 2^16).  So a mask is a function of (seed, offset, i) alone and is computed again by the backward pass
// instead of being stored.  Sixteen bits and not 32: rates then count in steps of 2^-16, and the scale 2^16 / (2^16 - threshold)
// makes up for the rounded rate, so that the expectation is exact.  With 32 bits and 10 rounds a pass over 64 Mi bf16 values took 72 us
// for the integer multiplications alone, with 16 bits 49 us, without a generator 44 us.
struct Drop {
    const long long* rng;       // {seed, offset} on the device; never null, dropout or none
    int on;                     // 0: no dropout
    unsigned limit;             // threshold * 2^16 - 1: a piece in the upper half of a word, lower half whatever it is, is kept iff word > limit
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
// The words that hold the pieces of elements i0 .. i0 + V - 1 (i0 a multiple of V) in their upper halves.
template <int V>
__device__ __forceinline__ void drop_pieces(const DropKey& k, unsigned long long i0, unsigned (&piece)[V]) {
    const uint4 w = drop_words(k, i0 >> 3);
    if constexpr (V == 8) {
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) piece[j] = (j & 1) ? u[j >> 1] : u[j >> 1] << 16;
    } else {
        const bool second = (i0 & 4) != 0;                          // of the block's two halves
        const unsigned u[2] = {second ? w.z : w.x, second ? w.w : w.y};
        if constexpr (V == 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j) piece[j] = (j & 1) ? u[j >> 1] : u[j >> 1] << 16;
        } else {
            const unsigned word = (i0 & 2) != 0 ? u[1] : u[0];
            if constexpr (V == 2) {
                piece[0] = word << 16;
                piece[1] = word;
            } else {
                piece[0] = (i0 & 1) != 0 ? word : word << 16;
            }
        }
    }
}
// Bit j: element i0 + j is kept.
template <int V>
__device__ __forceinline__ unsigned drop_mask(const Drop& d, const DropKey& k, unsigned long long i0) {
    unsigned piece[V], mask = 0;
    drop_pieces<V>(k, i0, piece);
#pragma unroll
    for (int j = 0; j < V; ++j) mask |= (piece[j] > d.limit ? 1u : 0u) << j;
    return mask;
}
// Scaled where it is kept, 0 where not (whatever the value was, a NaN included).
template <int V>
__device__ __forceinline__ Lanes<V> drop_masked(const Drop& d, unsigned mask, const Lanes<V>& v) {
    float f[V];
    mul(v, filled<V>(d.scale)).get(f);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = (mask >> j & 1u) ? f[j] : 0.f;
    return lanes<V>(f);
}
template <int V>
__device__ __forceinline__ Lanes<V> drop(const Drop& d, const DropKey& k, unsigned long long i0, const Lanes<V>& v) {
    unsigned piece[V];
    drop_pieces<V>(k, i0, piece);
    float f[V];
    mul(v, filled<V>(d.scale)).get(f);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = piece[j] > d.limit ? f[j] : 0.f;
    return lanes<V>(f);
}

// threshold and scale of a rate in [0, 1]; false outside (a NaN included).  Rate 1 keeps nothing.  Where nothing is dropped the kernels hold
// `idle` (two words on the device) in the place of rng, which may be null then: as with PARAM_ONE, no kernel holds a pointer that it must not
// follow, wherever the compiler moves the load to.
inline bool make_drop(double rate, const long long* rng, const long long* idle, Drop* d) {
    if (!(rate >= 0.0 && rate <= 1.0)) return false;
    const unsigned threshold = (unsigned)(rate * 65536.0 + 0.5);
    d->limit = threshold * 65536u - 1u;             // 65536 * 65536 wraps around to 0: no word is above the limit
    d->scale = threshold < 65536u ? (float)(65536.0 / (65536.0 - (double)threshold)) : 0.f;
    d->on = threshold > 0;                          // a threshold of 0 keeps every element as it is
    d->rng = d->on ? rng : idle;
    return true;
}

}  // namespace linf
