// Dropout of one tensor, or of a (value, lower, upper) triple under one mask, with a mask that is computed from (seed, offset,
// element number) and never stored.  The backward pass of dropout is dropout of the gradient under the same (seed, offset).
//
// Bound by HBM: each value is read once and written once.  A thread takes the 8 elements of one generator block, so the
// generator's seven rounds are paid once for 8 elements (and once for the 24 of a triple).  Measured on one B200: 64 x 256 x 64 x 64 bf16, value and
// gradient, 98 us, 5.5 TB/s (135 us with a multiplication by a kept scale or 0 for each tensor instead of one selection).
#include "vec.cuh"

namespace linf {
namespace {

struct Tensors { const void* in[3]; void* out[3]; };

// 8 elements as one or two 16-byte accesses
template <typename T> struct Eight {
    static constexpr int W = 16 / (int)sizeof(T);
    static __device__ __forceinline__ void load(const T* p, float (&f)[8]) {
#pragma unroll
        for (int h = 0; h < 8 / W; ++h) {
            float g[W];
            unpack<T, W>(load_once<T, W>(p + h * W), g);
#pragma unroll
            for (int j = 0; j < W; ++j) f[h * W + j] = g[j];
        }
    }
    static __device__ __forceinline__ void store(T* p, const float (&f)[8]) {
#pragma unroll
        for (int h = 0; h < 8 / W; ++h) {
            float g[W];
#pragma unroll
            for (int j = 0; j < W; ++j) g[j] = f[h * W + j];
            store_once<T, W>(p + h * W, pack<T, W>(g));
        }
    }
};

template <typename T, bool WIDE, int TENSORS>
__global__ void __launch_bounds__(256)
dropout_kernel(Tensors t, long long n, Drop d) {
    const DropKey key = drop_key(d);
    const long long step = (long long)gridDim.x * blockDim.x;
    for (long long b = (long long)blockIdx.x * blockDim.x + threadIdx.x; b * 8 < n; b += step) {
        const bool whole = WIDE && b * 8 + 8 <= n;
        float f[TENSORS][8];
        if (whole) {
#pragma unroll
            for (int k = 0; k < TENSORS; ++k) Eight<T>::load(static_cast<const T*>(t.in[k]) + b * 8, f[k]);
        } else {
#pragma unroll
            for (int k = 0; k < TENSORS; ++k)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (b * 8 + j < n) f[k][j] = to_float<T>(static_cast<const T*>(t.in[k])[b * 8 + j]);
        }
        unsigned piece[8];
        drop_pieces<8>(key, (unsigned long long)b * 8, piece);
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int k = 0; k < TENSORS; ++k) f[k][j] = piece[j] > d.limit ? f[k][j] * d.scale : 0.f;
        if (whole) {
#pragma unroll
            for (int k = 0; k < TENSORS; ++k) Eight<T>::store(static_cast<T*>(t.out[k]) + b * 8, f[k]);
        } else {
#pragma unroll
            for (int k = 0; k < TENSORS; ++k)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (b * 8 + j < n) static_cast<T*>(t.out[k])[b * 8 + j] = from_float<T>(f[k][j]);
        }
    }
}

__global__ void dropout_next_kernel(long long* state, unsigned long long replica, long long* used) {
    // an odd multiple of the replica's number: seeds of their own for 2^64 replicas, and that of the state for replica 0
    used[0] = (long long)((unsigned long long)state[0] + replica * 0x9E3779B97F4A7C15ull);
    used[1] = (long long)atomicAdd(reinterpret_cast<unsigned long long*>(state + 1), 1ull);
}

template <typename T, int TENSORS>
int launch(const Tensors& t, long long n, const Drop& d, cudaStream_t st) {
    bool wide = true;
    for (int k = 0; k < TENSORS; ++k) wide = wide && aligned16(t.in[k]) && aligned16(t.out[k]);
    const long long blocks = (n + 8 * 256 - 1) / (8 * 256), most = (long long)sm_count() * 64;
    const int grid = (int)(blocks < most ? blocks : most);
    if (wide) dropout_kernel<T, true, TENSORS><<<grid, 256, 0, st>>>(t, n, d);
    else dropout_kernel<T, false, TENSORS><<<grid, 256, 0, st>>>(t, n, d);
    return launch_status();
}
template <typename T>
int launch(const Tensors& t, int tensors, long long n, const Drop& d, cudaStream_t st) {
    return tensors == 1 ? launch<T, 1>(t, n, d, st) : tensors == 2 ? launch<T, 2>(t, n, d, st) : launch<T, 3>(t, n, d, st);
}

}  // namespace

int dropout(const void* const* in, void* const* out, int tensors, long long n, int type, double rate, const long long* rng, cudaStream_t st) {
    Drop d;
    if (!make_drop(rate, rng, nullptr, &d)) return LINF_ERR_RATE;
    if (!d.on) {                                     // nothing is dropped: every element as it is, a NaN's bits included
        for (int k = 0; k < tensors; ++k)
            if (out[k] != in[k] &&
                cudaMemcpyAsync(out[k], in[k], (size_t)n * (type == LINF_F32 ? 4 : 2), cudaMemcpyDeviceToDevice, st) != cudaSuccess)
                return LINF_ERR_LAUNCH;
        return LINF_OK;
    }
    Tensors t = {};
    for (int k = 0; k < tensors; ++k) { t.in[k] = in[k]; t.out[k] = out[k]; }
    if (type == LINF_F32) return launch<float>(t, tensors, n, d, st);
    if (type == LINF_F16) return launch<__half>(t, tensors, n, d, st);
    return launch<__nv_bfloat16>(t, tensors, n, d, st);
}

int dropout_next(long long* state, long long replica, long long* used, cudaStream_t st) {
    dropout_next_kernel<<<1, 1, 0, st>>>(state, (unsigned long long)replica, used);
    return launch_status();
}

}  // namespace linf
