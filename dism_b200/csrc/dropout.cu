// Dropout from a counter-based generator, with the residual addition: y = residual + x * keep * scale.
//
// Element i of the flattened tensor is kept when its 16-bit random number is at least `threshold` = round(65536 p), and
// scale = 65536 / (65536 - threshold) makes the kept part unbiased for that very threshold.  The numbers are the eight halves
// of one Philox4x32-10 block (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011)
// with the seed as its key and (i / 8, site, offset) as its counter.  The mask is a function of (seed, offset, site, i): nothing
// of it is stored, the backward of a call is the same call on the gradient without a residual, and neither the grid nor the
// vector width changes it.  Seed and offset are read from device memory when the kernel runs, so a captured graph draws new
// masks after the program has advanced the offset.
//
// 42 million bf16 elements, forward with a residual and backward: 98 us for both, 0.66 of the measured copy rate.  Neither side is
// saturated: 61 and 65 % of the issue slots, DRAM at 51 and 35 %; stalls are loads first, then the arithmetic pipes.  A grid that fills
// the device once and loads a block ahead was slower (65 + 52 us against 57.6 + 45.5 between events).
#include <cuda_fp16.h>

#include "dism_common.cuh"

namespace dism {
namespace {

constexpr int DROPOUT_THREADS = 256;

__device__ __forceinline__ uint4 philox(uint4 x, unsigned k0, unsigned k1) {
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t first = uint64_t(0xD2511F53u) * x.x, second = uint64_t(0xCD9E8D57u) * x.z;
        x = make_uint4(unsigned(second >> 32) ^ x.y ^ k0, unsigned(second), unsigned(first >> 32) ^ x.w ^ k1, unsigned(first));
        k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
    }
    return x;
}

template <typename T>
__device__ __forceinline__ float widen(T x) { return float(x); }
template <>
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T narrow(float x) { return T(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow(float x) { return __float2bfloat16(x); }
template <>
__device__ __forceinline__ __half narrow(float x) { return __float2half(x); }

template <typename T>
struct alignas(16) Eight {
    T x[8];
};

// VECTOR: all pointers are 16-byte aligned and whole blocks of eight move as 16-byte accesses.
template <typename T, bool RESIDUAL, bool VECTOR>
__global__ void __launch_bounds__(DROPOUT_THREADS) dropout_kernel(const T* __restrict__ x, const T* __restrict__ residual, int64_t count,
                                                                  unsigned threshold, float scale, const int64_t* __restrict__ seed,
                                                                  unsigned site, T* __restrict__ out) {
    const int64_t block = int64_t(blockIdx.x) * DROPOUT_THREADS + threadIdx.x, first = block * 8;
    if (first >= count) return;
    const int64_t key = __ldg(seed), offset = __ldg(seed + 1);
    const bool whole = VECTOR && first + 8 <= count;
    Eight<T> value, sum;
    if (whole) {
        value = *reinterpret_cast<const Eight<T>*>(x + first);
        if (RESIDUAL) sum = *reinterpret_cast<const Eight<T>*>(residual + first);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (first + i >= count) break;
            value.x[i] = x[first + i];
            if (RESIDUAL) sum.x[i] = residual[first + i];
        }
    }
    const uint4 r = philox(make_uint4(unsigned(block), site, unsigned(offset), unsigned(offset >> 32)), unsigned(key), unsigned(key >> 32));
    const unsigned words[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned number = i & 1 ? words[i / 2] >> 16 : words[i / 2] & 0xffffu;
        float y = number >= threshold ? widen(value.x[i]) * scale : 0.f;
        if (RESIDUAL) y += widen(sum.x[i]);
        value.x[i] = narrow<T>(y);
    }
    if (whole) {
        *reinterpret_cast<Eight<T>*>(out + first) = value;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (first + i < count) out[first + i] = value.x[i];
    }
}

template <typename T>
cudaError_t launch(const void* x, const void* residual, int64_t count, unsigned threshold, float scale, const int64_t* seed, unsigned site,
                   void* out, cudaStream_t stream) {
    const bool vector = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    auto* kernel = residual ? (vector ? dropout_kernel<T, true, true> : dropout_kernel<T, true, false>)
                            : (vector ? dropout_kernel<T, false, true> : dropout_kernel<T, false, false>);
    const int64_t per_block = 8 * DROPOUT_THREADS;
    KernelTimer timer("dropout", stream);
    kernel<<<unsigned((count + per_block - 1) / per_block), DROPOUT_THREADS, 0, stream>>>(
        static_cast<const T*>(x), static_cast<const T*>(residual), count, threshold, scale, seed, site, static_cast<T*>(out));
    return cudaGetLastError();
}
}  // namespace

cudaError_t launch_dropout(int type, const void* x, const void* residual, int64_t count, unsigned threshold, float scale,
                           const int64_t* seed, unsigned site, void* out, cudaStream_t stream) {
    if (type == 0) return launch<float>(x, residual, count, threshold, scale, seed, site, out, stream);
    if (type == 1) return launch<__half>(x, residual, count, threshold, scale, seed, site, out, stream);
    return launch<__nv_bfloat16>(x, residual, count, threshold, scale, seed, site, out, stream);
}

}  // namespace dism
