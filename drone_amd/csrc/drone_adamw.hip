// drone_adamw.hip — one AdamW step over many tensors with the clip by the global norm of their gradients:
//   norm = sqrt(sum g^2);  c = min(1, max_norm / (norm + 1e-6));  g' = c g
//   m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
// Two launches whatever the number of tensors (up to kAdamwTensors): the norm's partial sums (and the step counter, in HBM
// so that a captured step replays with an advancing t), then the update; one launch of one workgroup where all the tensors
// together are a few chunks (the six tensors of a 20-64-64-4 policy: 7.8 us, 9.6 in two). Everything in 32 bits; a 16-bit
// weight is its 32-bit master rounded once, and the master is what the next step starts from unless the weight is no longer
// that. Bound by memory: 21e6 16-bit weights with masters, 672 MB, 23 + 114 us (4.9 TB/s; a copy reaches 5.1; the norm has to
// have read every gradient before the first update, and reads them from the cache's leavings again).
#include <hip/hip_runtime.h>

#include "drone_policy.hpp"

#include "../../include/drone_vec.h"

namespace drone {
namespace {

constexpr int kThreads = 256;
constexpr int kSmallThreads = 1024;

// Which of the launch's tensors holds a chunk: every lane of the wave looks at one first_chunk of the table.
__device__ __forceinline__ int tensor_of(const AdamwArgs& a, int chunk) {
    const int lane = threadIdx.x & 63;
    const unsigned long long mine = __ballot(lane < a.count && a.t[lane < a.count ? lane : 0].first_chunk <= chunk);
    return __builtin_amdgcn_readfirstlane(__popcll(mine) - 1);
}

template <class T>
__device__ __forceinline__ void load8(const T* p, long long i, long long n, bool vec, float* f) {
    if (vec && i + 8 <= n) {
        struct Eight { T e[8]; };
        const Eight v = *(const Eight*)__builtin_assume_aligned(p + i, 16);
#pragma unroll
        for (int k = 0; k < 8; k++) f[k] = (float)v.e[k];
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) f[k] = i + k < n ? (float)p[i + k] : 0.f;
    }
}

template <class T>
__device__ __forceinline__ void store8(T* p, long long i, long long n, bool vec, const float* f) {
    if (vec && i + 8 <= n) {
        struct Eight { T e[8]; } v;
#pragma unroll
        for (int k = 0; k < 8; k++) v.e[k] = (T)f[k];
        *(Eight*)__builtin_assume_aligned(p + i, 16) = v;
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) if (i + k < n) p[i + k] = (T)f[k];
    }
}

__device__ __forceinline__ float block_sum(float v, float* join) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) join[threadIdx.x >> 6] = v;
    __syncthreads();
    return join[0] + join[1] + join[2] + join[3];
}

// 1 - b^t from log b, to a few 2^-24 of itself for every t (a power in 64 bits took 3 us of a small step).
__device__ __forceinline__ float correction(float log_b, int t) { return -expm1f(log_b * (float)t); }

// partial[0..1]: the two bias corrections of this step; partial[2 + k]: the sums of squares
template <class T>
__global__ __launch_bounds__(kThreads) void adamw_norm_kernel(AdamwArgs a) {
    __shared__ float join[4];
    if (a.advance && blockIdx.x == 0 && threadIdx.x == 0) {
        const int t = *a.step + 1;
        *a.step = t;
        a.partial[0] = correction(a.log_b1, t);
        a.partial[1] = correction(a.log_b2, t);
        if (a.norm && !a.chunks) *a.norm = 0.f;  // no gradients at all
    }
    if (!a.parts) return;
    // 64 bits: a thread of the largest calls adds up 131 072 squares (in 32, 2 048 equal ones were rounded alike, 9e-6 off)
    double sum = 0;
    for (int chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
        const AdamwTensor& t = a.t[tensor_of(a, chunk)];
        float g[8];
        load8((const T*)t.g, (long long)(chunk - t.first_chunk) * kAdamwChunk + threadIdx.x * 8, t.n, t.vec, g);
        float eight = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++) eight += g[k] * g[k];
        sum += eight;
    }
    const float all = block_sum((float)sum, join);
    if (threadIdx.x == 0) a.partial[2 + a.part0 + blockIdx.x] = all;
}

// What an element's update needs besides its own values: the clip, lr / (1 - b1^t) and 1 / (1 - b2^t). The update's square
// root and reciprocal are the hardware's (1 ulp each): correctly rounded ones, three an element, kept one workgroup's vector
// units busy for 7 us of a 5 764-weight step.
struct Step { float clip, rate, unbias; };

// The hardware's square root takes a denormal number for 0: v of gradients around 1e-19 is scaled into the normal ones and back.
// (Its reciprocal does so too, but eps is normal, and what is added to it no less.)
__device__ __forceinline__ float root(float v) {
    const bool low = v < 0x1p-96f;
    return __builtin_amdgcn_sqrtf(low ? v * 0x1p64f : v) * (low ? 0x1p-32f : 1.f);
}

// Eight elements and their state: asked for in one go, updated, stored.
template <class T>
struct Eight {
    float g[8], m[8], v[8], p[8];
    __device__ __forceinline__ void load(const AdamwTensor& t, long long i) {
        load8((const T*)t.g, i, t.n, t.vec, g);
        load8(t.m, i, t.n, t.vec, m);
        load8(t.v, i, t.n, t.vec, v);
        load8((const T*)t.p, i, t.n, t.vec, p);
        if (sizeof(T) == 4) return;
        // A 16-bit weight that is not its rounded master has been written since the last step (a loaded state, a target's
        // copy): the step starts from it. The two bytes more cost 21e6 weights 8 us (135 against 127).
        float master[8];
        load8(t.master, i, t.n, t.vec, master);
#pragma unroll
        for (int k = 0; k < 8; k++) p[k] = (float)(T)master[k] == p[k] ? master[k] : p[k];
    }
    __device__ __forceinline__ void step(const AdamwArgs& a, const Step& s) {
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float d = g[k] * s.clip;
            m[k] = a.b1 * m[k] + a.rest1 * d;
            v[k] = a.b2 * v[k] + a.rest2 * d * d;
            p[k] = p[k] * a.decay - s.rate * m[k] * __builtin_amdgcn_rcpf(root(v[k] * s.unbias) + a.eps);
        }
    }
    __device__ __forceinline__ void store(const AdamwTensor& t, long long i) const {
        store8(t.m, i, t.n, t.vec, m);
        store8(t.v, i, t.n, t.vec, v);
        if (sizeof(T) == 2) store8(t.master, i, t.n, t.vec, p);
        store8((T*)t.p, i, t.n, t.vec, p);
    }
};

__device__ __forceinline__ float clip_of(const AdamwArgs& a, float norm) {
    if (!(a.max_norm > 0.f)) return 1.f;
    return norm != norm ? norm : fminf(a.max_norm / (norm + 1e-6f), 1.f);  // fminf drops a NaN; a step on NaN gradients has to show
}

template <class T>
__global__ __launch_bounds__(kThreads) void adamw_update_kernel(AdamwArgs a) {
    __shared__ float join[4];
    const int chunk = blockIdx.x;
    const AdamwTensor& t = a.t[tensor_of(a, chunk)];
    const long long i = (long long)(chunk - t.first_chunk) * kAdamwChunk + threadIdx.x * 8;
    Eight<T> e;
    e.load(t, i);
    float clip = 1.f;
    if (a.parts) {  // every workgroup joins the partial sums in the same order
        float sum = 0.f;
        for (int k = threadIdx.x; k < a.parts; k += kThreads) sum += a.partial[2 + k];
        const float norm = sqrtf(block_sum(sum, join));
        clip = clip_of(a, norm);
        if (a.norm && chunk == 0 && threadIdx.x == 0 && a.advance) *a.norm = norm;
    }
    e.step(a, {clip, a.lr / a.partial[0], 1.f / a.partial[1]});
    e.store(t, i);
}

// The whole step in one workgroup: thread group `threadIdx.x / kThreads` has every fourth chunk, all of it in registers
// before the norm is joined, so the step takes one trip to memory.
template <class T>
__global__ __launch_bounds__(kSmallThreads) void adamw_small_kernel(AdamwArgs a) {
    constexpr int kGroups = kSmallThreads / kThreads, kMine = kAdamwSmall / kGroups;
    __shared__ float join[kSmallThreads / 64];
    const int group = threadIdx.x / kThreads, at = threadIdx.x % kThreads * 8;
    const int step = *a.step + 1;
    Eight<T> e[kMine];
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < kMine; k++) {
        const int chunk = group + k * kGroups;
        if (chunk >= a.chunks) break;
        const AdamwTensor& t = a.t[tensor_of(a, chunk)];
        e[k].load(t, (long long)(chunk - t.first_chunk) * kAdamwChunk + at);
    }
    const float c1 = correction(a.log_b1, step), c2 = correction(a.log_b2, step);
#pragma unroll
    for (int k = 0; k < kMine; k++)
        if (group + k * kGroups < a.chunks)
#pragma unroll
            for (int j = 0; j < 8; j++) sum += e[k].g[j] * e[k].g[j];
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if ((threadIdx.x & 63) == 0) join[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < kSmallThreads / 64; k++) sum += join[k];
    const float norm = sqrtf(sum);
    if (threadIdx.x == 0) {
        *a.step = step;  // (everyone has read it: the barrier)
        if (a.norm) *a.norm = norm;
    }
    const Step s = {clip_of(a, norm), a.lr / c1, 1.f / c2};
#pragma unroll
    for (int k = 0; k < kMine; k++) {
        const int chunk = group + k * kGroups;
        if (chunk >= a.chunks) break;
        const AdamwTensor& t = a.t[tensor_of(a, chunk)];
        e[k].step(a, s);
        e[k].store(t, (long long)(chunk - t.first_chunk) * kAdamwChunk + at);
    }
}

}  // namespace

int adamw_norm_launch(int dtype, const AdamwArgs& a, int blocks, hipStream_t s) {
    if (dtype == DRONE_F32) adamw_norm_kernel<float><<<blocks, kThreads, 0, s>>>(a);
    else if (dtype == DRONE_BF16) adamw_norm_kernel<__bf16><<<blocks, kThreads, 0, s>>>(a);
    else adamw_norm_kernel<_Float16><<<blocks, kThreads, 0, s>>>(a);
    return (int)hipGetLastError();
}

int adamw_update_launch(int dtype, const AdamwArgs& a, hipStream_t s) {
    if (!a.chunks) return 0;
    if (dtype == DRONE_F32) adamw_update_kernel<float><<<a.chunks, kThreads, 0, s>>>(a);
    else if (dtype == DRONE_BF16) adamw_update_kernel<__bf16><<<a.chunks, kThreads, 0, s>>>(a);
    else adamw_update_kernel<_Float16><<<a.chunks, kThreads, 0, s>>>(a);
    return (int)hipGetLastError();
}

int adamw_small_launch(int dtype, const AdamwArgs& a, hipStream_t s) {
    if (dtype == DRONE_F32) adamw_small_kernel<float><<<1, kSmallThreads, 0, s>>>(a);
    else if (dtype == DRONE_BF16) adamw_small_kernel<__bf16><<<1, kSmallThreads, 0, s>>>(a);
    else adamw_small_kernel<_Float16><<<1, kSmallThreads, 0, s>>>(a);
    return (int)hipGetLastError();
}

}  // namespace drone
